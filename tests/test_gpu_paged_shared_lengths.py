"""GPU parity of paged_sdpa over a shared prefix whose length is no multiple of 32,
with float64 attention over what the pages hold: who shares goes by the length as
given. Requests that begin inside it hold keys of their own, also those that begin
in the block that the length cuts."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from tests.paged_util import i32, rows
from tests.test_gpu_paged_shared import check

pytestmark = pytest.mark.gpu


def batch(rng, shared, starts, n, D, H, page, bits):
    """A cache whose requests that begin behind `shared` hold the same keys there, in
    the same pages (the last of them only in part, so each has a copy of that one);
    the others' pages are all their own. Returns (cache, table)."""
    width = -(-(max(starts) + max(n)) // page)
    common = shared // page
    cache = PagedKVCache(common + len(starts) * width, H, D, page_size=page, bits=bits)
    table = common + np.arange(len(starts) * width, dtype=np.int32).reshape(-1, width)
    behind = [s >= shared for s in starts]
    table[behind, :common] = np.arange(common)
    table = i32(table)
    k, v = rows(rng, shared, H, D), rows(rng, shared, H, D)
    for b, (s, m) in enumerate(zip(starts, n)):
        row = table[b:b + 1].contiguous()
        if behind[b]:
            cache.write(k, v, row, i32([0]))
            own, at = s + m - shared, shared
        else:
            own, at = s + m, 0
        cache.write(rows(rng, own, H, D), rows(rng, own, H, D), row, i32([at]))
    return cache, table


CASES = [   # shared, starts, new tokens; query heads, kv heads, head dim, page, bits
    (2050, [2048, 2060, 2100], [1, 1, 1], 8, 2, 128, 64, 16),          # the first is inside, in the cut block
    (2050, [2060, 2049, 2050, 2047], [1, 1, 1, 1], 8, 2, 128, 64, 8),  # a later one, and exactly behind
    (2079, [2050, 2049, 2048, 2078], [1, 1, 1, 1], 4, 1, 64, 32, 16),  # nobody shares
    (1055, [1024, 1055, 1100, 1054, 1300], [4, 4, 4, 4, 4], 10, 2, 128, 32, 16),
    (1111, [1088, 1111, 1200, 1110], [2, 1, 3, 1], 6, 1, 256, 64, 16),
    (1111, [1110, 1200, 1111, 1088], [2, 1, 3, 1], 6, 1, 256, 64, 8),
    (4101, [4100, 4200, 4101, 4096, 4130, 4300, 4099, 4150], [9, 8, 8, 30, 1, 7, 8, 9], 5, 1, 128, 64, 8),   # several tiles
]


@pytest.mark.parametrize("shared,starts,n,Hq,H,D,page,bits", CASES)
def test_requests_that_begin_in_the_cut_block(gpu, shared, starts, n, Hq, H, D, page, bits):
    rng = np.random.default_rng(shared + D + bits)
    cache, table = batch(rng, shared, starts, n, D, H, page, bits)
    q = rows(rng, sum(n), Hq, D)
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    lengths = [s + m for s, m in zip(starts, n)]
    got = paged_sdpa(q, cache, table, i32(starts), off, max_rows=max(n), shared=shared)
    check(cache, table, q, n, lengths, got, what=f"shared={shared}", rows_of=lambda m: [0, m - 1] if m > 1 else [0])
    if len(set(n)) == 1:
        check(cache, table, q, n, lengths, paged_sdpa(q, cache, table, i32(starts), shared=shared), what="equal rows",
              rows_of=lambda m: [0])
    cache.check_status()


def test_captured_steps_across_the_cut_block(gpu):
    """A captured step replayed as batches change under it: who shares is read from the
    positions, so a slot may hold a request of its own keys in one replay and one that
    shares in the next."""
    rng = np.random.default_rng(12)
    shared, n, Hq, H, D, page = 2050, 2, 8, 2, 128, 64
    batches = [[2048, 2060, 2100], [2300, 2049, 2050], [2047, 2048, 2049], [2050, 2051, 2100]]
    made = []
    for starts in batches:
        made.append(batch(rng, shared, [*starts, 2300], [n] * 4, D, H, page, 16))   # (the fourth: one width for all)
    cache = PagedKVCache(made[0][0].num_pages, H, D, page_size=page)
    table, start, q = made[0][1][:3].clone(), i32(batches[0]), rows(rng, 3 * n, Hq, D)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = paged_sdpa(q, cache, table, start, shared=shared)
    for _ in range(2):
        for (c, t), starts in zip(made, batches):
            cache.k_pages.copy_(c.k_pages)
            cache.v_pages.copy_(c.v_pages)
            table.copy_(t[:3])
            start.copy_(i32(starts))
            q.copy_(rows(rng, 3 * n, Hq, D))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            check(c, table, q, [n] * 3, [s + n for s in starts], out, what=str(starts))
            assert torch.equal(out, paged_sdpa(q, c, t[:3].contiguous(), start, shared=shared))
