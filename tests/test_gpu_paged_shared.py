"""GPU parity of paged_sdpa over a shared prefix with float64 attention over
what the pages hold, within the bounds that its roundings allow
(tests/paged_util.py)."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import head_norms, rotary_table
from oracle import paged as O
from tests.paged_util import attention_bound, check_rows, i32, num, rows, stored

pytestmark = pytest.mark.gpu


def batch(rng, prefix, tails, D, H, page, bits, poison=True):
    """A cache whose requests hold the same first `prefix` keys, in the pages
    that those fill whole, and tails[b] more; other places of the pool hold NaN
    if they can. Returns (cache, table, positions shared)."""
    common = prefix // page
    own = [-(-(prefix + t) // page) - common for t in tails]
    pages = common + sum(own) + 2
    order = rng.permutation(pages)
    table = np.full((len(tails), common + max(1, max(own))), -1, np.int32)
    table[:, :common] = order[:common]
    at = common
    for b, n in enumerate(own):
        table[b, common:common + n] = order[at:at + n]
        at += n
    table = torch.from_numpy(table).cuda()
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    if poison:
        if bits == 16:
            c.k_pages.fill_(float("nan"))
            c.v_pages.fill_(float("nan"))
        else:
            c.k_scales.fill_(float("nan"))
            c.v_scales.fill_(float("inf"))
    k, v = rows(rng, max(prefix, 1), H, D), rows(rng, max(prefix, 1), H, D)
    for b, t in enumerate(tails):
        if prefix:
            c.write(k, v, table[b:b + 1].contiguous(), i32([0]))
        if t:
            c.write(rows(rng, t, H, D), rows(rng, t, H, D), table[b:b + 1].contiguous(), i32([prefix]))
    return c, table, common * page


def check(c, table, q, n, lengths, got, what="", rows_of=None):
    lo = 0
    for b, (m, e) in enumerate(zip(n, lengths)):
        if m:
            k, v = stored(c, table, b, e)
            for at in ([slice(0, m)] if rows_of is None else [slice(i, i + 1) for i in rows_of(m)]):
                r = slice(lo + at.start, lo + at.stop)
                o, spread, reach = O.attend(num(q[r]), k, v, e - m + at.start)
                check_rows(num(got[r]), o, attention_bound(o, spread, reach, c.head_dim), f"{what} request {b} {at}")
        lo += m


CASES = [  # prefix, tail of each (its new tokens among it), new tokens; query heads, kv heads, head dim, page, bits
    (2048, [1, 1], [1, 1], 8, 8, 128, 64, 16), (2240, [5, 40, 300], [1, 1, 1], 40, 8, 128, 64, 8),
    (1025, [4, 9, 100, 33], [4, 1, 0, 3], 10, 2, 128, 32, 16), (1100, [7, 1, 2, 90], [2, 1, 2, 1], 5, 1, 64, 32, 8),
    (2000, [3] * 33, [1] * 33, 4, 1, 64, 64, 16), (2080, [8, 600], [8, 8], 4, 1, 256, 32, 16),
    (1100, [2, 5, 64, 33], [2, 5, 1, 1], 6, 1, 256, 64, 8), (1056, [20] * 70, [4] * 70, 10, 2, 128, 32, 16),
    (3000, [6, 9], [1, 1], 32, 1, 128, 128, 16), (4500, [90, 1, 31, 32, 33], [1, 1, 1, 1, 1], 2, 2, 128, 96, 8),
    # several tiles of 32 rows a request
    (4128, [50, 9, 8, 300, 31, 32, 33, 100], [8, 9, 8, 1, 0, 10, 12, 7], 5, 1, 128, 64, 16),
    (4100, [200, 64, 1, 70, 33, 40, 41, 42, 50], [30, 33, 1, 20, 33, 4, 5, 6, 7], 4, 1, 64, 64, 8),
    (4096, [41] * 8, [8] * 8, 32, 1, 128, 32, 8), (4160, [90, 300, 20, 20, 20, 20, 20, 20], [17] * 8, 2, 2, 256, 32, 16),
    # too short, or too many rows, to be worth a pass of its own
    (512, [50, 9], [50, 9], 5, 1, 128, 64, 16), (576, [200, 64, 1], [1, 3, 1], 4, 2, 64, 64, 8),
]


@pytest.mark.parametrize("prefix,tails,n,Hq,H,D,page,bits", CASES)
def test_matches_float64(gpu, prefix, tails, n, Hq, H, D, page, bits):
    rng = np.random.default_rng(prefix + sum(tails) + D + bits)
    c, table, shared = batch(rng, prefix, tails, D, H, page, bits)
    lengths = [prefix + t for t in tails]
    q = rows(rng, sum(n), Hq, D)
    start = i32([e - m for e, m in zip(lengths, n)])
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    got = paged_sdpa(q, c, table, start, off, max_rows=max(n), shared=shared)
    check(c, table, q, n, lengths, got)
    assert torch.equal(got, paged_sdpa(q, c, table, start, off, max_rows=max(n), shared=shared))
    # whole blocks of 32 are shared, whatever is said
    cut = max(1, shared - 7)
    check(c, table, q, n, lengths, paged_sdpa(q, c, table, start, off, max_rows=max(n), shared=cut), what="cut")
    check(c, table, q, n, lengths, paged_sdpa(q, c, table, start, off, shared=shared), what="no max_rows")
    if len(set(n)) == 1:
        assert torch.equal(paged_sdpa(q, c, table, start, shared=shared), got)
    c.check_status()


def test_more_rows_than_announced(gpu):
    """max_rows costs time, not results: too small for one request, or for all."""
    rng = np.random.default_rng(41)
    for D, bits in ((128, 16), (64, 8), (256, 16)):
        n, tails = [2, 45, 1, 90], [300, 45, 41, 120]
        c, table, shared = batch(rng, 1024, tails, D, 2, 64, bits)
        lengths = [1024 + t for t in tails]
        q = rows(rng, sum(n), 8, D)
        start, off = i32([e - m for e, m in zip(lengths, n)]), i32(np.concatenate([[0], np.cumsum(n)]))
        for max_rows in (1, 2, 8, 45, 1000):
            got = paged_sdpa(q, c, table, start, off, max_rows=max_rows, shared=shared)
            check(c, table, q, n, lengths, got, what=f"max_rows={max_rows}")


def test_many_requests(gpu):
    """More heads than workgroups for the tails."""
    rng = np.random.default_rng(42)
    tails = [1 + 7 * i % 90 for i in range(300)]
    c, table, shared = batch(rng, 1024, tails, 64, 4, 64, 16, poison=False)
    q = rows(rng, 300, 4, 64)
    got = paged_sdpa(q, c, table, i32([1023 + t for t in tails]), shared=shared)
    check(c, table, q, [1] * 300, [1024 + t for t in tails], got)


@pytest.mark.parametrize("bits", [8, 16])
def test_long_prefixes(gpu, bits):
    rng = np.random.default_rng(5 + bits)
    for prefix, tails, n, Hq, H in ((20000, [700, 30, 40, 1], [1, 9, 1, 1], 10, 2), (9000, [64] * 40, [4] * 40, 16, 2)):
        c, table, shared = batch(rng, prefix, tails, 128, H, 64, bits)
        lengths = [prefix + t for t in tails]
        q = rows(rng, sum(n), Hq, 128)
        off = i32(np.concatenate([[0], np.cumsum(n)]))
        got = paged_sdpa(q, c, table, i32([e - m for e, m in zip(lengths, n)]), off, max_rows=max(n), shared=shared)
        check(c, table, q, n, lengths, got, what=str(prefix),
              rows_of=lambda m: [0, m - 1] if m > 1 else [0])


def test_requests_that_begin_inside(gpu):
    """A request whose tokens lie in the prefix sees what is before them and no
    more; rows of nobody stay as they are; positions before the first key."""
    rng = np.random.default_rng(7)
    for bits, many in ((16, 1), (8, 1), (16, 60)):
        c, table, shared = batch(rng, 1024, [40, 70, 70, 70], 128, 2, 64, bits)
        n = [2, 3, many, 1]
        starts = [1024 + 30, 1000, 500, -3]
        q = rows(rng, sum(n) + 4, 8, 128)
        out = torch.full_like(q, 3.0)
        off = i32(np.concatenate([[0], np.cumsum(n)]))
        got = paged_sdpa(q, c, table, i32(starts), off, max_rows=max(n), shared=shared, out=out)
        assert (got[sum(n):] == 3).all() and (got[sum(n) - 1] == 0).all()
        lo = 0
        for b, m in enumerate(n[:3]):
            k, v = stored(c, table, b, starts[b] + m)
            o, spread, reach = O.attend(num(q[lo:lo + m]), k, v, starts[b])
            check_rows(num(got[lo:lo + m]), o, attention_bound(o, spread, reach, 128), f"request {b}")
            lo += m
        # exactly behind it, and no tokens at all
        one = paged_sdpa(q[:2], c, table[:2].contiguous(), i32([1024, 1023]), shared=shared)
        for b, s in enumerate((1024, 1023)):
            k, v = stored(c, table, b, s + 1)
            o, spread, reach = O.attend(num(q[b:b + 1]), k, v, s)
            check_rows(num(one[b:b + 1]), o, attention_bound(o, spread, reach, 128), f"at {s}")
        out.fill_(3.0)
        paged_sdpa(q, c, table, i32(starts), i32([0] * 5), max_rows=4, shared=shared, out=out)
        assert (out == 3).all()
        # rows that do not begin at the first, offsets that fall: nothing outside is touched
        paged_sdpa(q, c, table, i32([1060] * 4), i32([3, 4, 4, 5, 6]), max_rows=1, shared=shared, out=out)
        assert (out[:3] == 3).all() and (out[6:] == 3).all()
        k, v = stored(c, table, 2, 1061)
        o, spread, reach = O.attend(num(q[4:5]), k, v, 1060)
        check_rows(num(out[4:5]), o, attention_bound(o, spread, reach, 128), "a later row")


@pytest.mark.parametrize("bits", [8, 16])
def test_absent_pages_and_odd_values(gpu, bits):
    rng = np.random.default_rng(8)
    c, table, shared = batch(rng, 2048, [40, 40], 128, 1, 64, bits)
    q = rows(rng, 2, 4, 128)
    t = table.clone()
    t[:, 3] = -1   # keys 192..255 of the prefix
    got = paged_sdpa(q, c, t, i32([2087, 2087]), shared=shared)
    assert int(c.status().item()) == 1
    c.status().zero_()
    keep = np.r_[0:192, 256:2088]
    for b in range(2):
        k, v = (x[:, keep] for x in stored(c, table, b, 2088))
        o, spread, reach = O.attend(num(q[b:b + 1]), k, v, len(keep) - 1)
        check_rows(num(got[b:b + 1]), o, attention_bound(o, spread, reach, 128), f"request {b}")
    t[:] = -1
    assert (paged_sdpa(q, c, t, i32([2087, 2087]), shared=shared) == 0).all()
    c.status().zero_()
    # a value that is not a number: in the prefix all rows show it, in a tail its own
    bad = rows(rng, 1, 1, 128)
    bad[0, 0, 3] = float("nan")
    want = paged_sdpa(q, c, table, i32([2087, 2087]), shared=shared)
    c.write(torch.zeros_like(bad), bad, table[1:].contiguous(), i32([2074]))
    got = paged_sdpa(q, c, table, i32([2087, 2087]), shared=shared)
    assert torch.equal(got[0], want[0]) and torch.isnan(got[1, :, 3]).all()
    c.write(torch.zeros_like(bad), bad, table[:1].contiguous(), i32([100]))
    got = paged_sdpa(q, c, table, i32([2087, 2087]), shared=shared)
    assert torch.isnan(got[..., 3]).all()


def test_scores_of_minus_infinity(gpu):
    rng = np.random.default_rng(9)
    c, table, shared = batch(rng, 2048, [3, 3], 64, 1, 64, 16, poison=False)
    low = rows(rng, 2048, 1, 64)
    low[:, 0, 0] = float("-inf")
    q = rows(rng, 2, 2, 64).abs() + 0.5
    before = paged_sdpa(q, c, table, i32([2050, 2050]), shared=shared)
    c.write(low, rows(rng, 2048, 1, 64), table[:1].contiguous(), i32([0]))
    got = paged_sdpa(q, c, table, i32([2050, 2050]), shared=shared)
    for b in range(2):   # the prefix counts for nothing
        k, v = (x[:, 2048:] for x in stored(c, table, b, 2051))
        o, spread, reach = O.attend(num(q[b:b + 1]), k, v, 2)
        check_rows(num(got[b:b + 1]), o, attention_bound(o, spread, reach, 64), f"request {b}")
    c.write(low[:3], low[:3], table[:1].contiguous(), i32([2048]))
    got = paged_sdpa(q, c, table, i32([2050, 2050]), shared=shared)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all() and torch.isfinite(before).all()


@pytest.mark.parametrize("n,B", [(2, 2), (11, 8)])
def test_scores_of_every_size(gpu, n, B):
    """One key of the prefix or of the tail takes all; a maximum that rises or
    falls from the prefix to the tail."""
    rng = np.random.default_rng(10)
    prefix = 2048 if B == 2 else 4096
    tails = [100, 60, 33, 20, 64, 12, 99, 40][:B]
    for kind in ("large", "rising", "falling"):
        c, table, shared = batch(rng, prefix, tails, 128, 1, 32, 16, poison=False)
        keys = prefix + 100
        k, v = rows(rng, keys, 1, 128), rows(rng, keys, 1, 128)
        q = rows(rng, B * n, 4, 128)
        if kind == "large":
            k *= 20
            q *= 4
        else:
            ramp = torch.linspace(0, 30, keys, device="cuda")
            k[:, 0, 0] = (ramp if kind == "rising" else 30 - ramp).to(k.dtype)
            q[..., 0] = 40.0
        for b, t in enumerate(tails):
            c.write(k[:prefix + t], v[:prefix + t], table[b:b + 1].contiguous(), i32([0]))
        lengths = [prefix + t for t in tails]
        got = paged_sdpa(q, c, table, i32([e - n for e in lengths]), shared=shared)
        check(c, table, q, [n] * B, lengths, got, what=kind)


def test_decode_steps_and_graphs(gpu):
    """A batch as it is served: heads normalised, rotated and written, attended
    over the shared prefix, eagerly and captured; graphs of other row counts on
    the same stream replayed at once."""
    rng = np.random.default_rng(11)
    H, Hq, D, page, B = 2, 8, 128, 64, 5
    rot, norms = rotary_table(D, base=1e6), head_norms(*(torch.rand(D, device="cuda") + 0.5 for _ in range(2)))
    c, table, shared = batch(rng, 2048, [300] * B, D, H, page, 8)
    e = PagedKVCache(c.num_pages, H, D, page_size=page, bits=8)
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        getattr(e, name).copy_(getattr(c, name))
    start = i32([2100, 2048, 2200, 2060, 2150])
    parts = [tuple(rows(rng, B * n, h, D) for h in (Hq, H, H)) for n in (1, 4, 20)]

    def step(cache, q, k, v):
        turned = cache.write(k, v, table, start, queries=q, rotary=rot, norms=norms)
        return paged_sdpa(turned, cache, table, start, shared=shared)

    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in parts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(c, *p))
        graphs.append(g)
    for i in range(3):
        start.copy_(i32([2100 + i, 2048 + 3 * i, 2200 - i, 2060, 2150]))
        for g, out, p in zip(graphs, outs, parts):
            p[0].copy_(rows(rng, *p[0].shape))
            want = step(e, *p)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            n = p[0].shape[0] // B
            turned = e.write(p[1], p[2], table, start, queries=p[0], rotary=rot, norms=norms)
            check(e, table, turned, [n] * B, [int(s) + n for s in start], want, what=f"{n} rows",
                  rows_of=lambda m: [0, m - 1])
    # attention alone, replayed on streams at once
    graphs, outs, want = [], [], [paged_sdpa(p[0], c, table, start, shared=shared) for p in parts]
    torch.cuda.synchronize()
    for p in parts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_sdpa(p[0], c, table, start, shared=shared))
        graphs.append(g)
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)


def test_free_slots(gpu):
    """Slots of a batch without a request, the first one's among them: no rows, or
    a row of padding at position 0, and no pages."""
    rng = np.random.default_rng(15)
    for bits, B in ((16, 6), (8, 6), (16, 90)):
        busy = [2, 4, 5] if B == 6 else [70, 71, 89]
        c, own, shared = batch(rng, 2048, [40, 70, 9], 128, 2, 64, bits)
        table = torch.full((B, own.shape[1]), -1, dtype=torch.int32, device="cuda")
        table[busy] = own
        starts = np.zeros(B, np.int32)
        starts[busy] = [2087, 2117, 2056]
        q = rows(rng, B, 8, 128)
        for padded in (True, False):
            n = np.ones(B, np.int32) if padded else np.isin(np.arange(B), busy).astype(np.int32)
            off = np.concatenate([[0], np.cumsum(n)])
            out = paged_sdpa(q[:off[-1]], c, table, i32(starts), i32(off), max_rows=1, shared=shared)
            for i, b in enumerate(busy):
                k, v = stored(c, own, i, int(starts[b]) + 1)
                r = slice(off[b], off[b] + 1)
                o, spread, reach = O.attend(num(q[r]), k, v, int(starts[b]))
                check_rows(num(out[r]), o, attention_bound(o, spread, reach, 128), f"slot {b} of {B}")
            assert (out[off[:-1][np.isin(np.arange(B), busy, invert=True) & (n > 0)]] == 0).all()
            assert int(c.status().item()) == int(padded)   # (the padding's own positions have no page)
            c.status().zero_()
        # nobody lies behind it
        starts[:] = 5
        out = paged_sdpa(q, c, table, i32(starts), shared=shared)
        assert (out[[b for b in range(B) if b not in busy]] == 0).all()
        for i, b in enumerate(busy):
            k, v = stored(c, own, i, 6)
            o, spread, reach = O.attend(num(q[b:b + 1]), k, v, 5)
            check_rows(num(out[b:b + 1]), o, attention_bound(o, spread, reach, 128), f"inside, slot {b}")
        c.status().zero_()


def test_views_and_outputs(gpu):
    rng = np.random.default_rng(14)
    for n in (3, 50):
        c, table, shared = batch(rng, 2048, [80, 90], 64, 2, 32, 16)
        fused = rows(rng, 2 * n, 8 * 64)
        q = fused[:, :256].view(2 * n, 4, 64)
        start = i32([2128 - n, 2138 - n])
        want = paged_sdpa(q.contiguous(), c, table, start, scale=0.3, shared=shared)
        assert torch.equal(paged_sdpa(q, c, table.long(), start.cpu(), scale=0.3, shared=shared), want)
        wide = torch.zeros((2 * n, 8 * 64), dtype=torch.bfloat16, device="cuda")
        out = wide[:, 128:384].view(2 * n, 4, 64)
        paged_sdpa(q, c, table, start, scale=0.3, out=out, shared=shared)
        assert torch.equal(out, want) and (wide[:, :128] == 0).all() and (wide[:, 384:] == 0).all()
        paged_sdpa(q, c, table, start, scale=0.3, out=q, shared=shared)   # over its own queries
        assert torch.equal(q, want)


def test_refusals(gpu):
    c = PagedKVCache(4, 2, 64, page_size=32)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    table, start = i32([[0, 1], [0, 2]]), i32([40, 40])
    for kw in (dict(shared=-1), dict(shared=65), dict(shared=32, window=8)):
        with pytest.raises(ValueError):
            paged_sdpa(q, c, table, start, **kw)
    assert paged_sdpa(q[:0], c, table, start, shared=32).shape == (0, 4, 64)
