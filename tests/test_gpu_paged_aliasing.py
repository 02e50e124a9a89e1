"""Outputs of the paged operators laid over their inputs: the bits of the same
call with outputs of its own."""

import numpy as np
import pytest
import torch

from mtplx_amd._lib import MtpError
from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import apply_rotary, rotary_table
from tests.paged_util import i32, rows, tables

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


def test_write_and_attention_on_fused_rows(gpu):
    """Queries rotated, then attended, into columns beside them."""
    rng = np.random.default_rng(33)
    n, Hq, H, D, keys = 300, 8, 2, 128, 500
    table, pages = tables(rng, [keys], 64)
    a, b = (PagedKVCache(pages, H, D, page_size=64) for _ in range(2))
    rope, start = rotary_table(D, base=1e6), i32([keys - n])
    old = rows(rng, keys, H, D)
    for c in (a, b):
        c.write(old, old, table, i32([0]))
    fused = rows(rng, n, (2 * Hq + 2 * H) * D)
    q, k, v, out = (fused[:, lo * D:hi * D].view(n, hi - lo, D) for lo, hi in
                    ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H), (Hq + 2 * H, 2 * (Hq + H))))
    turned = a.write(k, v, table, start, queries=q, rotary=rope)
    want = paged_sdpa(turned, a, table, start)
    q0 = q.clone()
    assert b.write(k, v, table, start, queries=q, rotary=rope, out=out) is out
    assert torch.equal(out, turned) and torch.equal(q, q0) and torch.equal(a.k_pages, b.k_pages)
    b.write(k, v, table, start, queries=q, rotary=rope, out=q)
    assert torch.equal(q, turned)
    paged_sdpa(q, b, table, start, out=out)
    assert torch.equal(out, want) and torch.equal(q, turned)
    paged_sdpa(q, b, table, start, out=q)
    assert torch.equal(q, want)


def test_wide_index_arrays_do_not_wrap(gpu):
    """An int64 table on the GPU whose entries int32 cannot hold: no page of the
    pool is written or read through them."""
    rng = np.random.default_rng(34)
    c = PagedKVCache(4, 1, 64, page_size=32)
    x = rows(rng, 6, 1, 64)
    for entry in (2 ** 32, 2 ** 32 + 3, -2 ** 32 + 1):
        table = torch.tensor([[entry]], device="cuda")
        c.write(x, x, table, i32([0]))
        with pytest.raises(MtpError):
            c.check_status()
        assert not c.k_pages.any().item() and not c.v_pages.any().item()
        assert (paged_sdpa(x, c, table, i32([0])) == 0).all()
        with pytest.raises(MtpError):
            c.check_status()
    first = i32([[0]])
    c.write(x, x, first, torch.tensor([2 ** 32], device="cuda"))   # not position 0
    with pytest.raises(MtpError):
        c.check_status()
    assert not c.k_pages.any().item()
    c.write(x, x, first, i32([0]), torch.tensor([0, 2 ** 32 + 2], device="cuda"))   # past the rows: all six
    assert torch.equal(c.read(first, 6)[0][0, 0], x[:, 0])
    assert torch.equal(c.read(first, 6, lengths=torch.tensor([2 ** 32], device="cuda"))[0][0, 0], x[:, 0])


@pytest.mark.parametrize("n", [1, 4, 90])
def test_outputs_with_heads_outside_tokens(gpu, n):
    rng = np.random.default_rng(35)
    Hq, H, D, keys = 8, 2, 64, 200
    table, pages = tables(rng, [keys], 32)
    c = PagedKVCache(pages, H, D, page_size=32)
    old = rows(rng, keys, H, D)
    c.write(old, old, table, i32([0]))
    rope, start, pos = rotary_table(D, base=1e4), i32([keys - n]), i32(np.arange(keys - n, keys))
    q, k = rows(rng, n, Hq, D), rows(rng, n, H, D)
    out = lambda: torch.full((Hq, n + 1, D), 3.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for call in (lambda **kw: apply_rotary(rope, q, None, pos, **{a: (b, None) for a, b in kw.items()})[0],
                 lambda **kw: c.write(k, k, table, start, queries=q, rotary=rope, **kw),
                 lambda **kw: paged_sdpa(q, c, table, start, **kw),
                 lambda **kw: paged_sdpa(q, c, table, start, i32([0, n]), **kw)):
        want, buf = call(), out()
        got = call(out=buf[:, :n].transpose(0, 1))
        assert torch.equal(got, want) and torch.equal(buf[:, :n], want.transpose(0, 1)) and (buf[:, n] == 3).all()
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    want = apply_rotary(rope, q, None, pos)[0]
    apply_rotary(rope, turned, None, pos, out=(turned, None))
    assert torch.equal(turned, want)
