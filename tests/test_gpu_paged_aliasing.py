"""Outputs of the paged operators laid over their inputs: the bits of the same
call with outputs of its own."""

import numpy as np
import pytest
import torch

from mtplx_amd.rotary import apply_rotary, rotary_table
from tests.paged_util import i32, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,trad", [(128, False), (128, True), (24, False)])
def test_rotary_over_another_part(gpu, dims, trad):
    """Queries and keys that are one tensor, and outputs exchanged: many heads
    and tokens, so that a workgroup's items would meet."""
    rng = np.random.default_rng(31)
    T, H, D = 700, 24, 128
    t, pos = rotary_table(dims, base=1e5, traditional=trad), i32(rng.integers(0, 9000, T))
    q, k = rows(rng, T, H, D), rows(rng, T, H, D)
    wq, wk = apply_rotary(t, q, k, pos)
    x, y = q.clone(), torch.zeros_like(q)
    apply_rotary(t, x, x, pos, out=(x, y))
    assert torch.equal(x, wq) and torch.equal(y, wq)
    x = q.clone()
    apply_rotary(t, x, x, pos, out=(y.zero_(), x))
    assert torch.equal(x, wq) and torch.equal(y, wq)
    x, y = q.clone(), k.clone()
    apply_rotary(t, x, y, pos, out=(y, x))
    assert torch.equal(y, wq) and torch.equal(x, wk)
    x, y = q.clone(), k.clone()
    apply_rotary(t, x, y, pos, out=(x, y))
    assert torch.equal(x, wq) and torch.equal(y, wk)


def test_rotary_on_a_fused_projection(gpu):
    """In place on the parts of fused rows: no copy of either, the same bits,
    and the other columns stay."""
    rng = np.random.default_rng(32)
    T, Hq, H, D = 900, 16, 4, 128
    t, pos = rotary_table(D, base=1e6), i32(rng.integers(0, 9000, T))
    fused = rows(rng, T, (Hq + 2 * H) * D)
    q, k = fused[:, :Hq * D].view(T, Hq, D), fused[:, Hq * D:(Hq + H) * D].view(T, H, D)
    wq, wk = apply_rotary(t, q, k, pos)
    keep = fused[:, (Hq + H) * D:].clone()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    apply_rotary(t, q, k, pos, out=(q, k))
    assert torch.cuda.max_memory_allocated() == before
    assert torch.equal(q, wq) and torch.equal(k, wk) and torch.equal(fused[:, (Hq + H) * D:], keep)
