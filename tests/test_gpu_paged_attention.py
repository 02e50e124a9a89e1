"""GPU parity of paged_sdpa with float64 attention over what the pages hold,
within the bounds that its roundings allow (tests/paged_util.py)."""

import math

import numpy as np
import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import rotary_table
from oracle import paged as O
from tests.paged_util import attention_bound, check_rows, i32, num, rows, stored, tables

pytestmark = pytest.mark.gpu


def _filled(rng, lengths, D, H, page, bits, poison=True):
    """A cache whose requests hold `lengths` keys; the rest of the pool (other
    pages, the tails of the requests' last pages) holds NaN if it can."""
    table, pages = tables(rng, lengths, page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    if poison:
        if bits == 16:
            c.k_pages.fill_(float("nan"))
            c.v_pages.fill_(float("nan"))
        else:
            c.k_pages.fill_(113)
            c.v_pages.fill_(-101)
            c.k_scales.fill_(float("nan"))
            c.v_scales.fill_(float("inf"))
    for b, n in enumerate(lengths):
        if n:
            c.write(rows(rng, n, H, D), rows(rng, n, H, D), table[b:b + 1], i32([0]))
    return c, table


def _check(c, table, q, n, lengths, got, scale=None, what=""):
    """Rows of the requests (n[b] new tokens at the end of lengths[b] keys)."""
    lo = 0
    for b, (m, e) in enumerate(zip(n, lengths)):
        if m:
            k, v = stored(c, table, b, e)
            o, spread, reach = O.attend(num(q[lo:lo + m]), k, v, e - m, scale)
            check_rows(num(got[lo:lo + m]), o, attention_bound(o, spread, reach, c.head_dim), f"{what} request {b}")
        lo += m


CASES = [  # new tokens, keys in all; query heads, kv heads, head dim, page, bits
    ([1], [1], 1, 1, 128, 32, 16), ([1], [33], 40, 8, 128, 64, 16), ([1], [700], 5, 1, 64, 32, 8),
    ([1, 1, 1], [31, 32, 300], 4, 4, 128, 64, 8), ([4, 1, 3], [4, 129, 1000], 10, 2, 128, 64, 16),
    ([4, 0, 3], [64, 40, 1025], 8, 2, 128, 128, 8), ([8], [500], 4, 1, 256, 32, 16), ([2, 5], [90, 257], 6, 1, 256, 64, 8),
    ([1] * 80, [1 + 3 * i for i in range(80)], 2, 1, 64, 32, 16), ([32], [40], 1, 1, 128, 32, 16),
    ([1, 1], [2049, 5], 32, 1, 128, 64, 16),
    # chunks
    ([33], [33], 1, 1, 128, 32, 16), ([100], [100], 5, 1, 128, 64, 16), ([70], [333], 8, 2, 128, 64, 8),
    ([257, 1, 40], [257, 90, 400], 4, 2, 128, 64, 16), ([61, 0, 1, 1], [61, 7, 450, 9], 6, 2, 64, 32, 8),
    ([130], [700], 3, 1, 256, 64, 16), ([45, 80], [45, 600], 8, 1, 256, 32, 8), ([300], [300], 2, 2, 64, 96, 16),
    ([90], [91], 32, 1, 128, 32, 8), ([11], [700], 7, 1, 128, 256, 16),
]


@pytest.mark.parametrize("n,lengths,Hq,H,D,page,bits", CASES)
def test_matches_float64(gpu, n, lengths, Hq, H, D, page, bits):
    rng = np.random.default_rng(sum(n) * 31 + sum(lengths) + D + bits)
    c, table = _filled(rng, lengths, D, H, page, bits)
    T = sum(n)
    q = rows(rng, T, Hq, D)
    start = i32([e - m for e, m in zip(lengths, n)])
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    got = paged_sdpa(q, c, table, start, off, max_rows=max(n))
    _check(c, table, q, n, lengths, got)
    again = paged_sdpa(q, c, table, start, off, max_rows=max(n))
    assert torch.equal(got, again)
    other = paged_sdpa(q, c, table, start, off)   # the rows of the longest request unknown: the chunk kernel
    _check(c, table, q, n, lengths, other, what="no max_rows")
    if len(set(n)) == 1:
        assert torch.equal(paged_sdpa(q, c, table, start), got)
    c.check_status()


@pytest.mark.parametrize("bits", [8, 16])
def test_long_contexts_and_whole_prompts(gpu, bits):
    """Many workgroups to a row tile and many row tiles to a workgroup: a few
    rows of each against float64."""
    rng = np.random.default_rng(77 + bits)
    for n, lengths, Hq, H in (([4, 2], [30000, 777], 10, 2), ([64], [20001], 5, 1), ([2000, 900], [2000, 1900], 8, 2)):
        c, table = _filled(rng, lengths, 128, H, 64, bits)
        q = rows(rng, sum(n), Hq, 128)
        off = i32(np.concatenate([[0], np.cumsum(n)]))
        got = paged_sdpa(q, c, table, i32([e - m for e, m in zip(lengths, n)]), off, max_rows=max(n))
        assert torch.isfinite(got).all()
        lo = 0
        for b, (m, e) in enumerate(zip(n, lengths)):
            k, v = stored(c, table, b, e)
            for i in sorted({0, 1, m // 3, m // 2, m - 1} & set(range(m))):
                o, spread, reach = O.attend(num(q[lo + i:lo + i + 1]), k, v, e - m + i)
                check_rows(num(got[lo + i:lo + i + 1]), o, attention_bound(o, spread, reach, 128), f"{n} row {i}")
            lo += m


def test_scores_of_every_size(gpu):
    """Large scores (one key takes all), equal ones, and a running maximum that
    rises in every block."""
    rng = np.random.default_rng(2)
    for n, keys, Hq in ((1, 2000, 4), (60, 1500, 4)):
        for kind in ("large", "equal", "rising", "falling"):
            table, pages = tables(rng, [keys], 64)
            c = PagedKVCache(pages, 1, 128, page_size=64)
            k, v = rows(rng, keys, 1, 128), rows(rng, keys, 1, 128)
            q = rows(rng, n, Hq, 128)
            if kind == "large":
                k *= 20
                q *= 4
            elif kind == "equal":
                k[:] = k[:1]
            else:
                ramp = torch.linspace(0, 30, keys, device="cuda")
                k[:, 0, 0] = (ramp if kind == "rising" else 30 - ramp).to(k.dtype)
                q[..., 0] = 40.0
            c.write(k, v, table, i32([0]))
            got = paged_sdpa(q, c, table, i32([keys - n]))
            _check(c, table, q, [n], [keys], got, what=kind)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_row_depends_on_nothing_behind_it(gpu, few, bits):
    """NaN and infinities in later keys and values of the same request: earlier
    rows keep their bits, later ones show them."""
    rng = np.random.default_rng(21)
    n, keys, Hq = (4, 100, 4) if few else (90, 200, 4)
    c, table = _filled(rng, [keys], 128, 1, 64, bits)
    q = rows(rng, n, Hq, 128)
    want = paged_sdpa(q, c, table, i32([keys - n]))
    for at in (keys - 1, keys - 3):
        for value in (float("nan"), float("inf"), float("-inf")):
            for which in ("k", "v"):
                d = PagedKVCache(c.num_pages, 1, 128, page_size=64, bits=bits)
                for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                    if getattr(c, name) is not None:
                        getattr(d, name).copy_(getattr(c, name))
                bad = rows(rng, 1, 1, 128)
                bad[0, 0, 3] = value
                good = torch.zeros_like(bad)
                d.write(bad if which == "k" else good, bad if which == "v" else good, table, i32([at]))
                got = paged_sdpa(q, d, table, i32([keys - n]))
                first = at - (keys - n)
                assert torch.equal(got[:first], want[:first]), (at, value, which)
                if which == "v":
                    assert not torch.isfinite(got[first:, :, 3]).any()


def test_rows_without_keys_and_rows_of_nobody(gpu):
    rng = np.random.default_rng(3)
    for max_rows in (4, 0):
        c, table = _filled(rng, [64, 64, 64], 64, 1, 32, 16)
        q = rows(rng, 12, 2, 64)
        out = torch.full_like(q, 5.0)
        # request 0 begins two positions before its first key, request 1 has no rows, request 2 one
        r = paged_sdpa(q, c, table, i32([-2, 10, 63]), i32([1, 5, 5, 6]), max_rows=max_rows, out=out)
        assert r is out
        assert (out[0] == 5).all() and (out[6:] == 5).all() and (out[1:3] == 0).all()
        k, v = stored(c, table, 0, 64)
        o, spread, reach = O.attend(num(q[3:5]), k, v, 0)
        check_rows(num(out[3:5]), o, attention_bound(o, spread, reach, 64), "request 0")
        k, v = stored(c, table, 2, 64)
        o, spread, reach = O.attend(num(q[5:6]), k, v, 63)
        check_rows(num(out[5:6]), o, attention_bound(o, spread, reach, 64), "request 2")
        # no rows at all
        out.fill_(5.0)
        paged_sdpa(q, c, table, i32([0, 0, 0]), i32([3, 3, 3, 3]), max_rows=max_rows, out=out)
        assert (out == 5).all()
        # positions past the table: the keys that there are
        got = paged_sdpa(q[:3], c, table, i32([64, 100, 2 ** 31 - 1]), i32([0, 1, 2, 3]), max_rows=max_rows)
        for b in range(3):
            k, v = stored(c, table, b, 64)
            o, spread, reach = O.attend(num(q[b:b + 1]), k, v, 64)
            check_rows(num(got[b:b + 1]), o, attention_bound(o, spread, reach, 64), "past the table")
        assert int(c.status().item()) == 0


@pytest.mark.parametrize("bits", [8, 16])
def test_absent_pages(gpu, bits):
    """Keys without a page count as absent; the status says so."""
    rng = np.random.default_rng(13)
    for n in (2, 70):
        c, table = _filled(rng, [400], 128, 1, 64, bits)
        q = rows(rng, n, 4, 128)
        k, v = stored(c, table, 0, 400)
        t = table.clone()
        t[0, 1], t[0, 3] = -1, c.num_pages   # keys 64..127 and 192..255
        keep = np.r_[0:64, 128:192, 256:400]
        got = paged_sdpa(q, c, t, i32([400 - n]))
        with pytest.raises(_lib.MtpError):
            c.check_status()
        gone = 400 - len(keep)
        o, spread, reach = O.attend(num(q), k[:, keep], v[:, keep], 400 - gone - n)
        check_rows(num(got), o, attention_bound(o, spread, reach, 128), f"n={n}")
        t[:] = -1
        assert (paged_sdpa(q, c, t, i32([400 - n])) == 0).all()


def test_views_scale_and_outputs(gpu):
    rng = np.random.default_rng(14)
    for n in (3, 50):
        c, table = _filled(rng, [200], 64, 2, 32, 16)
        fused = rows(rng, n, 8 * 64)
        q = fused[:, :256].view(n, 4, 64)
        want = paged_sdpa(q.contiguous(), c, table, i32([200 - n]), scale=0.3)
        _check(c, table, q, [n], [200], want, scale=0.3)
        assert torch.equal(paged_sdpa(q, c, table.long(), torch.tensor([200 - n]), scale=0.3), want)
        wide = torch.zeros((n, 8 * 64), dtype=torch.bfloat16, device="cuda")
        out = wide[:, 128:384].view(n, 4, 64)
        paged_sdpa(q, c, table, i32([200 - n]), scale=0.3, out=out)
        assert torch.equal(out, want) and (wide[:, :128] == 0).all() and (wide[:, 384:] == 0).all()
        paged_sdpa(q, c, table, i32([200 - n]), scale=0.3, out=q)   # over its own queries
        assert torch.equal(q, want)


def test_shared_pages(gpu):
    """Two requests over one prefix: the same pages, read by both."""
    rng = np.random.default_rng(15)
    c = PagedKVCache(6, 2, 128, page_size=64)
    t = i32([[3, 1, 0], [3, 1, 5]])
    c.write(rows(rng, 128, 2, 128), rows(rng, 128, 2, 128), t[:1], i32([0]))
    c.write(rows(rng, 40, 2, 128), rows(rng, 40, 2, 128), t, i32([128, 128]))
    q = rows(rng, 40, 8, 128)
    _check(c, t, q, [20, 20], [148, 148], paged_sdpa(q, c, t, i32([128, 128])))


def test_refusals(gpu):
    c = PagedKVCache(2, 2, 64, page_size=32)
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    table, start = i32([[0], [1]]), i32([0, 0])
    for call in (lambda: paged_sdpa(q[:, :3], c, table, start), lambda: paged_sdpa(q[..., :32], c, table, start),
                 lambda: paged_sdpa(q[:3], c, table, start), lambda: paged_sdpa(q, c, table[0], start),
                 lambda: paged_sdpa(q, c, table, start[:1]), lambda: paged_sdpa(q, c, table, start, start),
                 lambda: paged_sdpa(q, c, table, start, scale=0.0), lambda: paged_sdpa(q, c, table, start, scale=-1.0),
                 lambda: paged_sdpa(q, c, table, start, scale=float("nan")),
                 lambda: paged_sdpa(q, c, table, start, out=q[:2]),
                 lambda: paged_sdpa(torch.zeros((4, 66, 64), dtype=torch.bfloat16, device="cuda"), c, table, start)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        paged_sdpa(q.half(), c, table, start)
    with pytest.raises(RuntimeError):
        paged_sdpa(q.cpu(), c, table, start)
    assert paged_sdpa(q[:0], c, table, start).shape == (0, 4, 64)


@pytest.mark.parametrize("bits", [8, 16])
def test_layers_written_and_attended(gpu, bits):
    """The operators as a decoder runs them: a prompt in chunks, then verify
    rows and decode rows of several requests, each call rotating, writing and
    attending; every output against float64 over all that was written."""
    rng = np.random.default_rng(30 + bits)
    H, Hq, D, page = 2, 8, 128, 32
    rot = rotary_table(D, base=1e6, scaling="yarn", factor=4.0, trained_positions=4096)
    table, pages = tables(rng, [300, 90, 200], page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    lengths = [0, 0, 0]
    for n in ([120, 40, 0], [77, 1, 64], [4, 4, 4], [1, 1, 1], [1, 0, 90]):
        T = sum(n)
        fused = rows(rng, T, (Hq + 2 * H) * D)
        q, k, v = (fused[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H)))
        off, start = i32(np.concatenate([[0], np.cumsum(n)])), i32(lengths)
        turned = c.write(k, v, table, start, off, max_rows=max(n), queries=q, rotary=rot)
        got = paged_sdpa(turned, c, table, start, off, max_rows=max(n))
        lengths = [e + m for e, m in zip(lengths, n)]
        _check(c, table, turned, n, lengths, got, what=str(n))
    c.check_status()


def test_streams_and_captured_steps(gpu):
    """Two captured steps that share a workspace, replayed in turn with eager
    calls of other sizes between them."""
    rng = np.random.default_rng(16)
    H, Hq, D, page, B = 2, 8, 128, 64, 3
    rot = rotary_table(D, base=1e6)
    table, pages = tables(rng, [4000] * B, page)
    c, e = (PagedKVCache(pages, H, D, page_size=page, bits=8) for _ in range(2))
    for b in range(B):
        k, v = rows(rng, 3900, H, D), rows(rng, 3900, H, D)
        for x in (c, e):
            x.write(k, v, table[b:b + 1], i32([0]))
    start = i32([3000, 50, 1700])
    parts = [tuple(rows(rng, B * n, h, D) for h in (Hq, H, H)) for n in (2, 40)]

    def step(cache, q, k, v):
        return paged_sdpa(cache.write(k, v, table, start, queries=q, rotary=rot), cache, table, start)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for p in parts:
            step(c, *p)   # workspaces
    side.synchronize()
    graphs, outs = [], []
    for p in parts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(c, *p))
        graphs.append(g)
    for i in range(4):
        start.copy_(i32([3000 + 11 * i, 50 + i, 1700 - 100 * i]))
        for g, out, p in zip(graphs, outs, parts):
            p[0].copy_(rows(rng, *p[0].shape))
            want = step(e, *p)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        got = step(c, *parts[1])
    side.synchronize()
    assert torch.equal(got, step(e, *parts[1]))


def test_captured_steps_at_once(gpu):
    """Steps captured on one stream hold workspaces of their own: replayed on
    two streams at the same time they give what they give in turn."""
    rng = np.random.default_rng(18)
    H, Hq, D, page, B = 2, 16, 128, 64, 2
    table, pages = tables(rng, [9000] * B, page)
    c = PagedKVCache(pages, H, D, page_size=page)
    for b in range(B):
        c.write(rows(rng, 9000, H, D), rows(rng, 9000, H, D), table[b:b + 1], i32([0]))
    start = i32([8900, 5000])
    qs = [rows(rng, B * n, Hq, D) for n in (4, 4, 100, 100)]
    want = [paged_sdpa(q, c, table, start) for q in qs]
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_sdpa(q, c, table, start))
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


def test_two_host_threads_on_one_stream(gpu):
    """Calls of two threads on the same stream share its workspace; each call's
    launches stay together."""
    import threading

    rng = np.random.default_rng(19)
    H, Hq, D, page = 2, 16, 128, 64
    table, pages = tables(rng, [6000], page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=8)
    c.write(rows(rng, 6000, H, D), rows(rng, 6000, H, D), table, i32([0]))
    qs = [rows(rng, n, Hq, D) for n in (2, 90)]
    start = i32([5900])
    want = [paged_sdpa(q, c, table, start) for q in qs]
    torch.cuda.synchronize()
    bad: list = []

    def work(q, w):
        for _ in range(60):
            bad.append(paged_sdpa(q, c, table, start).ne(w).any())

    threads = [threading.Thread(target=work, args=a) for a in zip(qs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(bad) == 120 and not any(bool(b) for b in bad)
