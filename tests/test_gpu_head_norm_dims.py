"""GPU parity of head norms at every head dim and every part of it that turns in
whole chunks, with the float64 oracle: each element of a head counts in its mean.
A mean without one chunk of eight of D elements would put the factor off by
about 4 / D, some 2^-6 at D = 256; the bound is that of
tests/test_gpu_head_norms.py, one rounding to bf16 and 2^-19.
"""

import numpy as np
import pytest
import torch

from mtplx_amd.rotary import apply_rotary, head_norms, rotary_table
from tests.paged_util import i32, rows
from tests.test_gpu_head_norms import check, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", range(8, 257, 8))
def test_every_part_that_turns(gpu, D):
    rng = np.random.default_rng(D)
    T = 3
    q, k = rows(rng, T, 3, D), rows(rng, T, 1, D)
    q[..., -8:] *= 4   # (the last chunk counts)
    wq, wk = weight(rng, D), weight(rng, D)
    pos = np.array([0, 77, 300000], np.int32)
    for dims in [*range(16, D, 16), D]:
        t = rotary_table(dims, base=1e6)
        qo, ko = apply_rotary(t, q, k, i32(pos), norms=head_norms(wq, wk, eps=1e-5))
        check(qo, q, wq, 1e-5, pos, t, f"q, {dims} of {D}")
        check(ko, k, wk, 1e-5, pos, t, f"k, {dims} of {D}")
        one = apply_rotary(t, q, k, i32(pos), norms=head_norms(wq, None, eps=1e-5))
        assert torch.equal(one[0], qo) and torch.equal(one[1], apply_rotary(t, q, k, i32(pos))[1]), dims


@pytest.mark.parametrize("D,dims", [(80, 32), (96, 64), (192, 128), (248, 240)])
def test_many_tokens_and_axes(gpu, D, dims):
    """Workgroups of two tokens, more heads than a round takes, in place, and
    positions of three axes."""
    rng = np.random.default_rng(D + dims)
    T = 1601
    fused = rows(rng, T, 14 * D)
    q, k = fused[:, :11 * D].view(T, 11, D), fused[:, 11 * D:].view(T, 3, D)
    w = weight(rng, D)
    t = rotary_table(dims, base=1e6, sections=(dims // 2 - 8, 4, 4))
    pos = rng.integers(0, 50000, (3, T)).astype(np.int32)
    want_q, want_k = q.clone(), k.clone()
    apply_rotary(t, q, k, i32(pos), norms=head_norms(w, w, eps=1e-5), out=(q, k))
    check(q, want_q, w, 1e-5, pos, t, "q")
    check(k, want_k, w, 1e-5, pos, t, "k")


def test_large_rows(gpu):
    """Squares that sum to nearly 2^128 are as any others; from there on the mean is
    infinite and the head zeros, its neighbours as they were."""
    rng = np.random.default_rng(3)
    D, T = 128, 4
    x = rows(rng, T, 2, D)
    x /= x.abs().amax(-1, keepdim=True)
    x[1] *= 2.0 ** 60
    x[2, 0] *= 2.0 ** 66
    x[3] *= 2.0 ** 100
    w = weight(rng, D)
    pos = np.arange(T, dtype=np.int32)
    for dims in (128, 64, 24):
        t = rotary_table(dims, base=1e6)
        got = apply_rotary(t, x, x[:, :1], i32(pos), norms=head_norms(w, w, eps=1e-5))
        check(got[0][:2], x[:2], w, 1e-5, pos[:2], t, "q")
        check(got[0][2:3, 1:], x[2:3, 1:], w, 1e-5, pos[2:3], t, "beside")
        check(got[1][:2], x[:2, :1], w, 1e-5, pos[:2], t, "k")
        assert (got[0][2, 0] == 0).all() and (got[0][3] == 0).all() and (got[1][2:] == 0).all()
