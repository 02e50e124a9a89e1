"""Paged writes on both sides of the rules that choose how a call's work is cut: a
block of keys by one wave or by eight, queries in the write's launch or in one of
their own. The bits are those of apply_rotary on the same rows and a plain write."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import apply_rotary, head_norms, rotary_table
from tests.paged_util import i32, rows, tables
from tests.test_gpu_head_norms import weight

pytestmark = pytest.mark.gpu


def written(rng, n, start, Hq, Hkv, D, bits, dims, normed, trad=False, padded=0):
    t = rotary_table(dims, base=1e6, traditional=trad)
    table, pages = tables(rng, [a + b for a, b in zip(start, n)], 64)
    T = sum(n) + padded
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    q, k, v = rows(rng, T, Hq, D), rows(rng, T, Hkv, D), rows(rng, T, Hkv, D)
    norms = head_norms(weight(rng, D), weight(rng, D)) if normed else None
    pos = i32(np.concatenate([*(s + np.arange(m) for s, m in zip(start, n)), np.zeros(padded, int)]))
    want_q, want_k = apply_rotary(t, q, k, pos, norms=norms)
    cache, plain = (PagedKVCache(pages, Hkv, D, page_size=64, bits=bits) for _ in range(2))
    out = torch.full_like(q, 3.0)
    cache.write(k, v, table, i32(start), off, queries=q, rotary=t, norms=norms, out=out)
    plain.write(want_k, v, table, i32(start), off)
    cache.check_status()
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        a, b = getattr(cache, name), getattr(plain, name)
        assert a is None or torch.equal(a, b), name
    assert torch.equal(out[:T - padded], want_q[:T - padded]) and (out[T - padded:] == 3).all()


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("D,Hkv,n", [(64, 2, 2000), (64, 2, 3000), (128, 2, 2900), (128, 2, 3700), (128, 2, 4500),
                                     (256, 4, 1400), (256, 4, 1900), (256, 4, 2300)])
@pytest.mark.parametrize("bits", [8, 16])
def test_blocks_of_keys(gpu, D, Hkv, n, bits, normed):
    written(np.random.default_rng(n + D + bits), [n], [5], 2 * Hkv, Hkv, D, bits, D, normed)


@pytest.mark.parametrize("T", [2000, 2100])
@pytest.mark.parametrize("dims,trad", [(64, False), (256, False), (256, True), (24, False)])
def test_queries_of_wide_heads(gpu, T, dims, trad):
    """24 heads of 256: 48 Ki rows of queries and more have a launch of their own;
    rows behind the last request stay as they are."""
    written(np.random.default_rng(T + dims), [T - 40, 3, 0, 30], [5, 90, 7, 0], 24, 4, 256, 16, dims, True, trad, padded=7)
