"""paged_sdpa over long shares of keys: every 32-key block counts exactly once.

A workgroup looks its page list up 64 blocks at a time, and a row tile's keys
are cut between workgroups; a block lost or counted twice at such a seam weighs
a thousandth of a long row. So the values mark the blocks: V is 1 in column
(block + 7 head) % D and 0 elsewhere, an output element is then the weight of
the few blocks of its column, and the bound (relative to that weight) is passed
by nothing that moves one of them.

All requests take their pages from one pool, each in an order of its own. The
reference is float64 on the GPU, over what the raw pages hold."""

import numpy as np
import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from oracle import paged as O
from tests.paged_util import HALF, i32, rows

pytestmark = pytest.mark.gpu


def _pool(rng, keys, D, H, page, bits):
    """A cache full of keys, its values marking their blocks."""
    pages = -(-keys // page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    n = pages * page
    v = torch.zeros((n, H, D), dtype=torch.bfloat16, device="cuda")
    block = torch.arange(n, device="cuda") // 32
    for h in range(H):
        v[torch.arange(n, device="cuda"), h, (block + 7 * h) % D] = 1.0
    c.write(rows(rng, n, H, D), v, torch.arange(pages, dtype=torch.int32, device="cuda")[None], i32([0]))
    return c


def _held(c, pages, scales, kind, ids, h):
    """float64 [positions, D] of head h in pages `ids`."""
    at = torch.from_numpy(O.page_order(kind, c.head_dim, c.bits).reshape(-1)).cuda()
    x = pages[ids, h].double()[..., at].reshape(-1, c.head_dim)
    return x if scales is None else x * scales[ids, h].double().reshape(-1, 1)


def _check(c, table, q, n, lengths, got, stride):
    """Rows of every stride-th token and the last, all heads."""
    D, H, rep = c.head_dim, c.n_kv_heads, q.shape[1] // c.n_kv_heads
    lo = 0
    for b, (m, e) in enumerate(zip(n, lengths)):
        if not m:
            continue
        toks = torch.tensor(sorted({*range(0, m, stride), m - 1}), device="cuda")
        there = (table[b] >= 0).repeat_interleave(c.page_size)[:e]
        ids = table[b].clamp(min=0)[:-(-e // c.page_size)].long()
        pos = (e - m + toks).repeat_interleave(rep)
        for h in range(H):
            k = _held(c, c.k_pages, c.k_scales, "k", ids, h)[:e]
            v = _held(c, c.v_pages, c.v_scales, "v", ids, h)[:e]
            x = q[lo + toks, h * rep:(h + 1) * rep].reshape(-1, D).double()
            s = x @ k.t() / D ** 0.5
            s = s.masked_fill((torch.arange(e, device="cuda") > pos[:, None]) | ~there, float("-inf"))
            p = torch.softmax(s, -1)
            o = p @ v   # (values are positive: also the spread)
            reach = (x.abs() @ k.abs().t()).amax(-1, keepdim=True) / D ** 0.5
            bound = (2.02 * HALF + 2 * reach * (D * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -14) * o
            y = got[lo + toks, h * rep:(h + 1) * rep].reshape(-1, D).double()
            bad = ~((y - o).abs() <= bound + 1e-30)
            assert not bad.any(), f"request {b}, head {h}: {int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"
        lo += m


def _run(c, rng, n, lengths, Hq, stride, absent, scale=0.2):
    """scale: queries small enough that no key takes all."""
    page = c.page_size
    t = np.full((len(n), max(-(-e // page) for e in lengths)), -1, np.int32)
    for b, e in enumerate(lengths):
        used = -(-e // page)
        t[b, :used] = rng.permutation(c.num_pages)[:used]
        if absent:   # one page, far in; every ninth; one near the end: lists that begin with, hold and end with one
            t[b, {0: [used * 5 // 8], 1: list(range(4, used, 9)), 2: [used - 2]}[b % 3]] = -1
    table = torch.from_numpy(t).cuda()
    q = rows(rng, sum(n), Hq, c.head_dim, scale=scale)
    off, start = i32(np.concatenate([[0], np.cumsum(n)])), i32([e - m for m, e in zip(n, lengths)])
    got = paged_sdpa(q, c, table, start, off, max_rows=max(n))
    _check(c, table, q, n, lengths, got, stride)
    if absent:
        with pytest.raises(_lib.MtpError):
            c.check_status()
    else:
        c.check_status()


@pytest.mark.parametrize("absent", [False, True])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_chunks_of_many_keys_a_workgroup(gpu, D, bits, absent):
    """5800 to 10800 keys a share: page lists are refilled, K and V slots go
    round many times."""
    rng = np.random.default_rng(50 + D + bits + absent)
    c = _pool(rng, 20100, D, 8, 96, bits)
    _run(c, rng, [300, 64, 200, 130], [15300, 20064, 9200, 17130], 32, 23, absent)


@pytest.mark.parametrize("absent", [False, True])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_of_many_keys_a_workgroup(gpu, D, bits, absent):
    """9400 to 18800 keys a share: a wave's page list is refilled."""
    rng = np.random.default_rng(60 + D + bits + absent)
    c = _pool(rng, 40010, D, 8, 96, bits)
    _run(c, rng, [4, 2, 3, 4] * 4, [40000, 33007, 38000, 39999] * 4, 32, 1, absent)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,lengths,Hq,H,stride", [
    ([4, 2], [30000, 777], 10, 2, 1), ([64], [20001], 5, 1, 7), ([2000, 900], [2000, 1900], 8, 2, 41),
    ([7, 0, 1, 61], [7000, 5, 300, 61], 12, 4, 1), ([1] * 9, [1 + 511 * i for i in range(9)], 8, 1, 1),
])
def test_seams_of_short_shares(gpu, n, lengths, Hq, H, stride, bits):
    rng = np.random.default_rng(sum(lengths) + bits)
    c = _pool(rng, max(lengths), 128, H, 64, bits)
    _run(c, rng, n, lengths, Hq, stride, False)
    _run(c, rng, n, lengths, Hq, stride, len(n) == 2)


@pytest.mark.parametrize("bits", [8, 16])
def test_pages_past_32_bit_offsets(gpu, bits):
    """The last pages of a pool of more than 2^31 elements: the bits of a small
    pool that holds the same."""
    D, H, page = 128, 8, 256
    pages = 2 ** 31 // (D * H * page) + 5
    rng = np.random.default_rng(70 + bits)
    big, small = (PagedKVCache(p, H, D, page_size=page, bits=bits) for p in (pages, 4))
    tables = [i32([[pages - 1, pages - 3, pages - 2, pages - 4]]), i32([[0, 1, 2, 3]])]
    k, v = rows(rng, 1000, H, D), rows(rng, 1000, H, D)
    for c, t in zip((big, small), tables):
        c.write(k, v, t, i32([0]))
    for n in (3, 200):
        q = rows(rng, n, 4 * H, D)
        want = paged_sdpa(q, small, tables[1], i32([1000 - n]))
        assert torch.isfinite(want).all() and torch.equal(paged_sdpa(q, big, tables[0], i32([1000 - n])), want)
    big.check_status()


@pytest.mark.parametrize("bits", [8, 16])
def test_hints_that_are_wrong(gpu, bits):
    """max_rows below or above the longest request: the same rows stored, the
    same attention within its bound."""
    rng = np.random.default_rng(80 + bits)
    n, lengths, Hq, H, D = [300, 1, 40], [900, 200, 40], 8, 2, 128
    c = _pool(rng, 900, D, H, 64, bits)
    used = [-(-e // 64) for e in lengths]
    t = np.full((3, max(used)), -1, np.int32)
    for b, u in enumerate(used):
        t[b, :u] = rng.permutation(c.num_pages)[:u]
    table, off = torch.from_numpy(t).cuda(), i32([0, 300, 301, 341])
    start = i32([e - m for m, e in zip(n, lengths)])
    q = rows(rng, 341, Hq, D, scale=0.2)
    for hint in (1, 2, 4, 7, 299, 5000, 0, -3, None):
        _check(c, table, q, n, lengths, paged_sdpa(q, c, table, start, off, max_rows=hint), 17)
    pools = [PagedKVCache(c.num_pages * 3, H, D, page_size=64, bits=bits) for _ in range(3)]
    apart = (table + i32([[0], [c.num_pages], [2 * c.num_pages]])).masked_fill(table < 0, -1).int()
    k, v = rows(rng, 341, H, D), rows(rng, 341, H, D)
    for p, hint in zip(pools, (300, 1, 9000)):
        p.write(k, v, apart, start, off, max_rows=hint)
        p.check_status()
        assert torch.equal(p.k_pages, pools[0].k_pages) and torch.equal(p.v_pages, pools[0].v_pages)
    c.check_status()
