"""GPU parity of paged_sdpa behind a sliding window, with first tokens that stay
visible, with float64 attention over what the pages hold, within the bounds
that its roundings allow (tests/paged_util.py)."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import head_norms, rotary_table
from oracle import paged as O
from tests.paged_util import attention_bound, check_rows, i32, num, rows, stored, tables
from tests.test_gpu_paged_attention import _filled

pytestmark = pytest.mark.gpu


def given_back(table, n, lengths, page, window, sinks):
    """The table without the pages that no new token sees."""
    t = table.clone()
    for b, (m, e) in enumerate(zip(n, lengths)):
        first = max(0, e - m - window + 1)
        for i in range(table.shape[1]):
            if i * page >= sinks and (i + 1) * page <= first:
                t[b, i] = -1
    return t


def check(c, table, q, n, lengths, got, window, sinks, what="", rows_of=None):
    lo = 0
    for b, (m, e) in enumerate(zip(n, lengths)):
        if m:
            k, v = stored(c, table, b, e)
            for at in ([slice(0, m)] if rows_of is None else [slice(i, i + 1) for i in rows_of(m)]):
                r = slice(lo + at.start, lo + at.stop)
                o, spread, reach = O.attend(num(q[r]), k, v, e - m + at.start, window=window, sinks=sinks)
                check_rows(num(got[r]), o, attention_bound(o, spread, reach, c.head_dim), f"{what} request {b} {at}")
        lo += m


CASES = [  # new tokens, keys in all; query heads, kv heads, head dim, page, bits; window, sinks
    ([1], [1], 1, 1, 128, 32, 16, 1, 0), ([1], [500], 40, 8, 128, 64, 16, 1, 0), ([1], [500], 40, 8, 128, 64, 16, 1, 1),
    ([1], [700], 5, 1, 64, 32, 8, 100, 4), ([1, 1, 1], [31, 32, 300], 4, 4, 128, 64, 8, 33, 5),
    ([4, 1, 3], [4, 129, 1000], 10, 2, 128, 64, 16, 64, 64), ([4, 0, 3], [64, 40, 1025], 8, 2, 128, 128, 8, 200, 31),
    ([8], [500], 4, 1, 256, 32, 16, 129, 3), ([2, 5], [90, 257], 6, 1, 256, 64, 8, 40, 100),
    ([1] * 80, [1 + 3 * i for i in range(80)], 2, 1, 64, 32, 16, 50, 2), ([32], [40], 1, 1, 128, 32, 16, 5, 3),
    ([1, 1], [2049, 5], 32, 1, 128, 64, 16, 2000, 33), ([4], [400], 4, 1, 128, 64, 16, 90, 320),
    # chunks
    ([33], [33], 1, 1, 128, 32, 16, 7, 0), ([100], [100], 5, 1, 128, 64, 16, 32, 1), ([70], [333], 8, 2, 128, 64, 8, 100, 64),
    ([257, 1, 40], [257, 90, 400], 4, 2, 128, 64, 16, 128, 4), ([61, 0, 1, 1], [61, 7, 450, 9], 6, 2, 64, 32, 8, 20, 40),
    ([130], [700], 3, 1, 256, 64, 16, 300, 7), ([45, 80], [45, 600], 8, 1, 256, 32, 8, 64, 0),
    ([300], [300], 2, 2, 64, 96, 16, 1, 2), ([90], [91], 32, 1, 128, 32, 8, 60, 90), ([11], [700], 7, 1, 128, 256, 16, 333, 50),
    ([600], [900], 4, 1, 128, 64, 16, 250, 96), ([500], [500], 8, 1, 64, 64, 8, 1000, 16), ([129], [400], 2, 1, 128, 32, 16, 65, 65),
]


@pytest.mark.parametrize("n,lengths,Hq,H,D,page,bits,window,sinks", CASES)
def test_matches_float64(gpu, n, lengths, Hq, H, D, page, bits, window, sinks):
    rng = np.random.default_rng(sum(n) * 31 + sum(lengths) + D + bits + window)
    c, table = _filled(rng, lengths, D, H, page, bits)
    q = rows(rng, sum(n), Hq, D)
    start = i32([e - m for e, m in zip(lengths, n)])
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    kept = given_back(table, n, lengths, page, window, sinks)
    got = paged_sdpa(q, c, kept, start, off, max_rows=max(n), window=window, sinks=sinks)
    check(c, table, q, n, lengths, got, window, sinks)
    assert torch.equal(got, paged_sdpa(q, c, table, start, off, max_rows=max(n), window=window, sinks=sinks))
    other = paged_sdpa(q, c, kept, start, off, window=window, sinks=sinks)   # the longest request unknown
    check(c, table, q, n, lengths, other, window, sinks, what="no max_rows")
    if len(set(n)) == 1:
        assert torch.equal(paged_sdpa(q, c, kept, start, window=window, sinks=sinks), got)
    c.check_status()   # pages given back were not asked for


def test_more_rows_than_announced(gpu):
    """max_rows costs time, not results: too small for one request, or for all."""
    rng = np.random.default_rng(41)
    for D, bits, window, sinks in ((128, 16, 70, 5), (64, 8, 300, 0), (256, 16, 40, 33)):
        n, lengths = [2, 45, 1, 90], [300, 200, 41, 90]
        c, table = _filled(rng, lengths, D, 2, 64, bits)
        q = rows(rng, sum(n), 8, D)
        start, off = i32([e - m for e, m in zip(lengths, n)]), i32(np.concatenate([[0], np.cumsum(n)]))
        for max_rows in (1, 2, 8, 45, 1000):
            got = paged_sdpa(q, c, table, start, off, max_rows=max_rows, window=window, sinks=sinks)
            check(c, table, q, n, lengths, got, window, sinks, what=f"max_rows={max_rows}")


def test_many_requests(gpu):
    """More heads than workgroups: each whole in one."""
    rng = np.random.default_rng(42)
    lengths = [1 + 7 * i % 400 for i in range(600)]
    c, table = _filled(rng, lengths, 64, 4, 64, 16, poison=False)
    q = rows(rng, 600, 4, 64)
    got = paged_sdpa(q, c, table, i32([e - 1 for e in lengths]), window=100, sinks=3)
    check(c, table, q, [1] * 600, lengths, got, 100, 3)


@pytest.mark.parametrize("bits", [8, 16])
def test_long_contexts_and_whole_prompts(gpu, bits):
    rng = np.random.default_rng(77 + bits)
    for n, lengths, Hq, H, window, sinks in (([4, 2], [30000, 777], 10, 2, 4096, 4), ([64], [20001], 5, 1, 1000, 64),
                                             ([2000, 900], [2000, 1900], 8, 2, 500, 0), ([4000], [4000], 4, 1, 128, 1)):
        c, table = _filled(rng, lengths, 128, H, 64, bits)
        q = rows(rng, sum(n), Hq, 128)
        off = i32(np.concatenate([[0], np.cumsum(n)]))
        got = paged_sdpa(q, c, given_back(table, n, lengths, 64, window, sinks),
                         i32([e - m for e, m in zip(lengths, n)]), off, max_rows=max(n), window=window, sinks=sinks)
        assert torch.isfinite(got).all()
        check(c, table, q, n, lengths, got, window, sinks, what=str(n),
              rows_of=lambda m: sorted({0, 1, m // 3, m // 2, m - 2, m - 1, *range(120, 136)} & set(range(m))))
        c.check_status()


@pytest.mark.parametrize("n,keys,Hq", [(3, 500, 4), (90, 500, 4), (300, 300, 8)])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_window_over_everything_is_none(gpu, n, keys, Hq, bits):
    rng = np.random.default_rng(keys + n)
    c, table = _filled(rng, [keys], 128, 2, 64, bits)
    q = rows(rng, n, Hq, 128)
    want = paged_sdpa(q, c, table, i32([keys - n]), window=keys)
    check(c, table, q, [n], [keys], want, None, 0)
    for window in (keys + 1, 2 ** 31 - 1, 2 ** 40):
        got = paged_sdpa(q, c, table, i32([keys - n]), window=window)
        check(c, table, q, [n], [keys], got, None, 0, what=f"window={window}")
    # and so are sinks that reach every row
    got = paged_sdpa(q, c, table, i32([keys - n]), window=3, sinks=2 ** 31 - 1)
    check(c, table, q, [n], [keys], got, None, 0)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("bits", [8, 16])
def test_hidden_keys_do_not_count(gpu, few, bits):
    """NaN, infinities and large numbers in keys and values behind the window
    (in the blocks that it reads, too): the rows that do not see them keep
    their bits, the others show them."""
    rng = np.random.default_rng(23)
    n, keys, Hq, window, sinks = (4, 300, 4, 70, 5) if few else (90, 400, 4, 70, 5)
    c, table = _filled(rng, [keys], 128, 1, 64, bits)
    q = rows(rng, n, Hq, 128)
    start = keys - n
    want = paged_sdpa(q, c, table, i32([start]), window=window, sinks=sinks)
    for at in (0, 4, 5, 6, 31, start - window, start - window + 1, start - window + 3, start - 1):
        for value in (float("nan"), float("inf"), float("-inf"), 2.0 ** 40):
            for which in ("k", "v"):
                d = PagedKVCache(c.num_pages, 1, 128, page_size=64, bits=bits)
                for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                    if getattr(c, name) is not None:
                        getattr(d, name).copy_(getattr(c, name))
                bad = rows(rng, 1, 1, 128)
                bad[0, 0, 3] = value
                good = torch.zeros_like(bad)
                d.write(bad if which == "k" else good, bad if which == "v" else good, table, i32([at]))
                got = paged_sdpa(q, d, table, i32([start]), window=window, sinks=sinks)
                pos = start + np.arange(n)
                seen = torch.from_numpy((at <= pos) & ((at > pos - window) | (at < sinks))).cuda()
                assert torch.equal(got[~seen], want[~seen]), (at, value, which)
                if which == "v" and not np.isfinite(value):
                    assert not torch.isfinite(got[seen][..., 3]).any(), (at, value)


def test_odd_positions_and_rows_of_nobody(gpu):
    rng = np.random.default_rng(3)
    for max_rows in (4, 0):
        c, table = _filled(rng, [64, 64, 64], 64, 1, 32, 16)
        q = rows(rng, 12, 2, 64)
        out = torch.full_like(q, 5.0)
        kw = dict(window=3, sinks=1)
        r = paged_sdpa(q, c, table, i32([-2, 10, 63]), i32([1, 5, 5, 6]), max_rows=max_rows, out=out, **kw)
        assert r is out and (out[0] == 5).all() and (out[6:] == 5).all() and (out[1:3] == 0).all()
        for b, lo, hi, at in ((0, 3, 5, 0), (2, 5, 6, 63)):
            k, v = stored(c, table, b, 64)
            o, spread, reach = O.attend(num(q[lo:hi]), k, v, at, **kw)
            check_rows(num(out[lo:hi]), o, attention_bound(o, spread, reach, 64), f"request {b}")
        # positions past the table: what the window leaves of the keys that there are
        starts = [64, 65, 2 ** 31 - 1]
        got = paged_sdpa(q[:3], c, table, i32(starts), i32([0, 1, 2, 3]), max_rows=max_rows, **kw)
        for b in range(3):
            k, v = stored(c, table, b, 64)
            o, spread, reach = O.attend(num(q[b:b + 1]), k, v, starts[b], **kw)
            check_rows(num(got[b:b + 1]), o, attention_bound(o, spread, reach, 64), "past the table")
        assert (paged_sdpa(q[:1], c, table[:1], i32([1000]), max_rows=max_rows, window=3) == 0).all()
        assert int(c.status().item()) == 0


@pytest.mark.parametrize("bits", [8, 16])
def test_absent_pages(gpu, bits):
    """A page that a row sees and that is not there counts as absent and sets the status."""
    rng = np.random.default_rng(13)
    for n in (2, 70):
        c, table = _filled(rng, [400], 128, 1, 64, bits)
        q = rows(rng, n, 4, 128)
        k, v = stored(c, table, 0, 400)
        t = table.clone()
        t[0, 4] = -1   # keys 256..319
        got = paged_sdpa(q, c, t, i32([400 - n]), window=200, sinks=10)
        assert int(c.status().item()) == 1
        c.status().zero_()
        nk = num(q)
        for i in range(n):
            p = 400 - n + i
            j = np.arange(p + 1)
            j = j[((j > p - 200) | (j < 10)) & ((j < 256) | (j >= 320))]
            o, spread, reach = O.attend(nk[i:i + 1], k[:, j], v[:, j], len(j) - 1)
            check_rows(num(got[i:i + 1]), o, attention_bound(o, spread, reach, 128), f"n={n} row {i}")
        t[:] = -1
        assert (paged_sdpa(q, c, t, i32([400 - n]), window=200, sinks=10) == 0).all()


def test_scores_of_minus_infinity(gpu):
    """A row all of whose visible scores are -infinity is NaN, as softmax is; one
    that sees another key is not."""
    rng = np.random.default_rng(31)
    for n in (2, 90):
        table, pages = tables(rng, [200], 64)
        c = PagedKVCache(pages, 1, 64, page_size=64)
        k, v = rows(rng, 200, 1, 64), rows(rng, 200, 1, 64)
        k[100:, 0, 0] = float("-inf")
        c.write(k, v, table, i32([0]))
        q = rows(rng, n, 2, 64).abs() + 0.5
        got = paged_sdpa(q, c, table, i32([200 - n]), window=20)
        p = np.arange(200 - n, 200)
        blind = torch.from_numpy(p - 19 >= 100).cuda()
        assert torch.isnan(got[blind]).all() and torch.isfinite(got[~blind]).all()
        assert torch.isfinite(paged_sdpa(q, c, table, i32([200 - n]), window=20, sinks=1)).all()


@pytest.mark.parametrize("bits", [8, 16])
def test_layers_written_and_attended(gpu, bits):
    """The operators as a windowed decoder runs them: heads normalised, rotated by
    three axes, written and attended, pages given back as the window leaves
    them; every output against float64 over all that was written."""
    rng = np.random.default_rng(30 + bits)
    H, Hq, D, page, window, sinks = 2, 8, 128, 32, 60, 4
    rot = rotary_table(D, base=1e6, sections=(16, 24, 24))
    norms = head_norms(*(torch.rand(D, device="cuda") + 0.5 for _ in range(2)))
    table, pages = tables(rng, [300, 90, 200], page)
    full = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    lengths = [0, 0, 0]
    for n in ([120, 40, 0], [77, 1, 64], [4, 4, 4], [1, 1, 1], [1, 0, 90]):
        T = sum(n)
        fused = rows(rng, T, (Hq + 2 * H) * D)
        q, k, v = (fused[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H)))
        off, start = i32(np.concatenate([[0], np.cumsum(n)])), i32(lengths)
        pos = torch.from_numpy(rng.integers(0, 9000, (3, T)).astype(np.int32)).cuda()
        lengths = [e + m for e, m in zip(lengths, n)]
        kept = given_back(table, n, lengths, page, window, sinks)
        turned = c.write(k, v, kept, start, off, max_rows=max(n), queries=q, rotary=rot, norms=norms, positions=pos)
        full.write(k, v, table, start, off, rotary=rot, norms=norms, positions=pos)
        got = paged_sdpa(turned, c, kept, start, off, max_rows=max(n), window=window, sinks=sinks)
        check(full, table, turned, n, lengths, got, window, sinks, what=str(n))
    c.check_status()


def test_captured_steps(gpu):
    """Windowed calls captured on one stream, replayed in turn and on two streams
    at once, with eager calls of other sizes between."""
    rng = np.random.default_rng(18)
    H, Hq, D, page, B = 2, 16, 128, 64, 2
    table, pages = tables(rng, [9000] * B, page)
    c = PagedKVCache(pages, H, D, page_size=page)
    for b in range(B):
        c.write(rows(rng, 9000, H, D), rows(rng, 9000, H, D), table[b:b + 1], i32([0]))
    start = i32([8000, 5000])
    qs = [rows(rng, B * n, Hq, D) for n in (1, 4, 100)]
    kw = dict(window=700, sinks=4)
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_sdpa(q, c, table, start, **kw))
        graphs.append(g)
    for i in range(3):
        start.copy_(i32([8000 + 13 * i, 5000 - 300 * i]))
        want = [paged_sdpa(q, c, table, start, **kw) for q in qs]
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w), i


def test_two_host_threads_on_one_stream(gpu):
    """Windowed calls of two threads on the same stream share its workspace."""
    import threading

    rng = np.random.default_rng(19)
    H, Hq, D, page = 2, 16, 128, 64
    table, pages = tables(rng, [6000], page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=8)
    c.write(rows(rng, 6000, H, D), rows(rng, 6000, H, D), table, i32([0]))
    qs = [rows(rng, n, Hq, D) for n in (2, 90)]
    start, kw = i32([5900]), dict(window=3000, sinks=4)
    want = [paged_sdpa(q, c, table, start, **kw) for q in qs]
    torch.cuda.synchronize()
    bad: list = []

    def work(q, w):
        for _ in range(40):
            bad.append(paged_sdpa(q, c, table, start, **kw).ne(w).any())

    threads = [threading.Thread(target=work, args=a) for a in zip(qs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(bad) == 80 and not any(bool(b) for b in bad)


def test_views_and_outputs(gpu):
    rng = np.random.default_rng(14)
    for n in (3, 50, 300):
        c, table = _filled(rng, [400], 64, 2, 32, 16)
        fused = rows(rng, n, 8 * 64)
        q = fused[:, :256].view(n, 4, 64)
        start, kw = i32([400 - n]), dict(scale=0.3, window=90, sinks=3)
        want = paged_sdpa(q.contiguous(), c, table, start, **kw)
        assert torch.equal(paged_sdpa(q, c, table.long(), torch.tensor([400 - n]), **kw), want)
        wide = torch.zeros((n, 8 * 64), dtype=torch.bfloat16, device="cuda")
        out = wide[:, 128:384].view(n, 4, 64)
        paged_sdpa(q, c, table, start, out=out, **kw)
        assert torch.equal(out, want) and (wide[:, :128] == 0).all() and (wide[:, 384:] == 0).all()
        paged_sdpa(q, c, table, start, out=q, **kw)   # over its own queries
        assert torch.equal(q, want)


def test_refusals(gpu):
    c = PagedKVCache(2, 2, 64, page_size=32)
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    table, start = i32([[0], [1]]), i32([0, 0])
    for kw in (dict(window=0), dict(window=-1), dict(window=4, sinks=-1), dict(sinks=1)):
        with pytest.raises(ValueError):
            paged_sdpa(q, c, table, start, **kw)
    assert paged_sdpa(q[:0], c, table, start, window=2).shape == (0, 4, 64)
