"""GPU parity of head norms and positions of several axes, alone
(``apply_rotary``) and on the way into the cache (``PagedKVCache.write``), with
the float64 oracle.

Bound. One rounding to bf16, 2^-8 of the value. Before it, in fp32: the sum of
D squares (chains of 8, then a tree: at most 13 roundings of 2^-24 relative,
halved by the root), its mean, sum, root and reciprocal (4), the two products
(2): 2^-20 of a normalised element; the rotation 2^-21 gain (|x1| + |x2|) as
without norms. Together at most 2^-19 gain (|x1| + |x2|) of normalised elements.
"""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import apply_rotary, head_norms, rotary_table
from oracle import paged as O
from tests.paged_util import HALF, check_rows, i32, num, rows, stored, tables

pytestmark = pytest.mark.gpu


def weight(rng, D, dtype=torch.bfloat16):
    return torch.from_numpy(np.exp(0.5 * rng.standard_normal(D)).astype(np.float32)).to("cuda", dtype)


def expected(x, w, eps, pos, t):
    """(float64 rows, their bound)."""
    y = num(x) if w is None else O.norm_heads(num(x), num(w), eps)
    axis = t.axis or np.zeros(t.dims // 2, int)
    want = O.rotate_axes(y, np.asarray(pos).reshape(t.axes, -1), axis, t.frequencies, t.dims, t.traditional, t.gain)
    a = np.abs(y)
    mate = a.copy()
    h = t.dims // 2
    i1, i2 = (np.arange(0, t.dims, 2), np.arange(1, t.dims, 2)) if t.traditional else (np.arange(h), np.arange(h) + h)
    mate[..., i1], mate[..., i2] = a[..., i2], a[..., i1]
    mate[..., t.dims:] = 0.0
    return want, HALF * np.abs(want) + max(1.0, abs(t.gain)) * 2.0 ** -19 * (a + mate)


def check(got, x, w, eps, pos, t, what):
    want, bound = expected(x, w, eps, pos, t)
    check_rows(num(got), want, bound, what)


def some_positions(rng, axes, T, far=300000):
    pos = rng.integers(-3, far, (axes, T)).astype(np.int32)
    return pos[0] if axes == 1 else pos


SHAPES = [   # T, Hq, Hkv, D, dims, traditional, sections, interleaved
    (1, 40, 8, 128, 128, False, None, False), (1, 1, 1, 64, 64, True, (16, 16), False),
    (3, 5, 1, 64, 32, False, (4, 6, 6), False), (17, 4, 2, 128, 96, True, (18, 15, 15), True),
    (33, 2, 2, 256, 256, False, (32, 48, 48), False), (100, 3, 1, 128, 24, False, (6, 3, 3), True),
    (5, 3, 1, 80, 20, True, None, False), (7, 2, 1, 64, 2, False, (1,), False), (9, 2, 2, 40, 6, True, (1, 1, 1), True),
    (13, 12, 12, 80, 80, False, (10, 10, 10, 10), True), (2, 3, 2, 8, 4, False, None, False),
    (513, 3, 1, 64, 64, False, (12, 10, 10), True), (2100, 2, 1, 64, 48, True, (9, 9, 6), False),
    (600, 24, 4, 256, 64, False, (12, 10, 10), True), (31, 1, 3, 256, 240, False, (120,), False),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,dims,trad,sections,turn", SHAPES)
def test_apply_rotary(gpu, T, Hq, Hkv, D, dims, trad, sections, turn):
    rng = np.random.default_rng(T * 1000 + D + dims)
    t = rotary_table(dims, base=1e6, traditional=trad, sections=sections, interleaved=turn, gain=1.25)
    assert list(t.axis or [0] * (dims // 2)) == O.pair_axes(dims // 2, sections, turn).tolist()
    q, k = rows(rng, T, Hq, D, scale=3.0), rows(rng, T, Hkv, D, scale=0.05)
    pos = some_positions(rng, t.axes, T)
    wq, wk = weight(rng, D), weight(rng, D, torch.float32)
    n = head_norms(wq, wk, eps=1e-5)
    on_gpu = torch.from_numpy(pos).cuda()
    qo, ko = apply_rotary(t, q, k, on_gpu, norms=n)
    check(qo, q, wq, 1e-5, pos, t, "q")
    check(ko, k, wk, 1e-5, pos, t, "k")
    # one side's norm, or none: the other side is as without
    plain = apply_rotary(t, q, k, on_gpu)
    for norms, a, b in ((head_norms(wq, None, eps=1e-5), qo, plain[1]), (head_norms(None, wk, eps=1e-5), plain[0], ko)):
        got = apply_rotary(t, q, k, on_gpu, norms=norms)
        assert torch.equal(got[0], a) and torch.equal(got[1], b)
    check(plain[0], q, None, 0.0, pos, t, "q, no norms")
    check(plain[1], k, None, 0.0, pos, t, "k, no norms")
    alone, none = apply_rotary(t, q, None, pos, norms=n)   # positions from the host
    assert none is None and torch.equal(alone, qo)


def test_equal_axes_are_one_position(gpu):
    """Text: all axes count alike, and the result has the bits of a table without axes."""
    rng = np.random.default_rng(3)
    T = 70
    q, k = rows(rng, T, 4, 128), rows(rng, T, 2, 128)
    pos = i32(rng.integers(0, 50000, T))
    n = head_norms(weight(rng, 128), weight(rng, 128))
    for kw in (dict(), dict(traditional=True), dict(dims=64)):
        dims = kw.pop("dims", 128)
        one = rotary_table(dims, base=1e6, **kw)
        for turn in (False, True):
            many = rotary_table(dims, base=1e6, sections=(dims // 2 - 20, 10, 10), interleaved=turn, **kw)
            a, b = apply_rotary(one, q, k, pos), apply_rotary(many, q, k, pos.expand(3, T))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            a, b = apply_rotary(one, q, k, pos, norms=n), apply_rotary(many, q, k, pos.expand(3, T), norms=n)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_table_that_does_not_turn(gpu):
    rng = np.random.default_rng(6)
    D = 128
    t = rotary_table(D, frequencies=[0.0] * (D // 2))
    x, w = rows(rng, 40, 3, D), weight(rng, D)
    got = apply_rotary(t, x, None, i32(range(40)), norms=head_norms(w, None))[0]
    want = O.norm_heads(num(x), num(w), 1e-6)
    check_rows(num(got), want, HALF * np.abs(want) + 2.0 ** -20 * np.abs(want), "norms alone")
    assert torch.equal(apply_rotary(t, x, None, i32(range(40)))[0], x)


def test_rows_of_odd_values(gpu):
    """Zeros, tiny and huge rows, one with a NaN, one with an infinity: each row
    alone decides its result."""
    rng = np.random.default_rng(4)
    D = 128
    t = rotary_table(64, base=1e4)
    x = rows(rng, 8, 2, D)
    x[1] = 0.0
    x[2] *= 2.0 ** -60
    x[3] *= 2.0 ** 50
    x[4, 0, 7] = float("nan")
    x[5, 1, 100] = float("inf")
    w = weight(rng, D)
    pos = np.arange(8, dtype=np.int32)
    got = apply_rotary(t, x, x[:, :1], i32(pos), norms=head_norms(w, w, eps=1e-6))[0]
    want, bound = expected(x, w, 1e-6, pos, t)
    sane = [0, 1, 2, 3, 6, 7]
    check_rows(num(got)[sane], want[sane], bound[sane], "rows")
    g = num(got)
    assert (g[1] == 0).all() and np.isnan(g[4, 0]).all() and np.isfinite(g[4, 1]).all()
    assert np.isnan(g[5, 1, 100]) and (np.delete(g[5, 1, 64:], 36) == 0).all() and np.isfinite(g[5, 0]).all()
    zero = apply_rotary(t, x, None, i32(pos), norms=head_norms(w, None, eps=0.0))[0]
    assert torch.isnan(zero[1]).all()   # 0 / sqrt(0), as the formula reads


def test_views_and_in_place(gpu):
    rng = np.random.default_rng(9)
    T, Hq, Hkv, D = 21, 4, 2, 64
    n = head_norms(weight(rng, D), weight(rng, D))
    for dims, trad in ((64, False), (24, False), (24, True), (32, False)):
        t = rotary_table(dims, base=1e4, traditional=trad, sections=(dims // 2 - 2, 1, 1))
        pos = torch.from_numpy(some_positions(rng, 3, T)).cuda()
        fused = rows(rng, T, (Hq + 2 * Hkv) * D)
        q = fused[:, :Hq * D].view(T, Hq, D)
        k = fused[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        want = apply_rotary(t, q.contiguous(), k.contiguous(), pos, norms=n)
        got = apply_rotary(t, q, k, pos, norms=n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # positions in another order of memory, and wide ones
        assert torch.equal(apply_rotary(t, q, k, pos.t().contiguous().t().long(), norms=n)[0], want[0])
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(apply_rotary(t, turned, k, pos, norms=n)[0], want[0])
        keep = fused.clone()
        r = apply_rotary(t, q, k, pos, norms=n, out=(q, k))
        assert r[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(fused[:, (Hq + Hkv) * D:], keep[:, (Hq + Hkv) * D:])


WRITES = [   # rows of each request, start of each, Hq, Hkv, D, bits, dims, traditional, sections, interleaved, page
    ([1], [0], 8, 8, 128, 16, 128, False, None, False, 64),
    ([1, 4, 2], [37, 100, 63], 5, 1, 64, 8, 64, False, (12, 10, 10), True, 32),
    ([70, 1, 33, 0, 5], [0, 500, 31, 7, 64], 10, 2, 128, 8, 128, False, (16, 24, 24), False, 64),
    ([100, 9], [3, 0], 6, 1, 256, 16, 64, False, (12, 10, 10), True, 64),
    ([40, 3], [10, 95], 4, 4, 64, 16, 48, True, (8, 8, 8), False, 32),
    ([45, 2], [0, 17], 4, 2, 128, 16, 24, False, (6, 3, 3), True, 128),
    ([45, 2], [0, 17], 4, 2, 256, 8, 256, True, None, False, 128),
    ([333], [0], 3, 3, 64, 8, 24, False, None, False, 32),
    ([2049, 3], [5, 0], 2, 1, 256, 16, 64, False, (12, 10, 10), True, 64),   # queries by a launch of their own
    ([2100], [0], 2, 1, 256, 8, 24, False, None, False, 64),
]


@pytest.mark.parametrize("n,start,Hq,Hkv,D,bits,dims,trad,sections,turn,page,normed",
                         [w + (normed,) for w in WRITES for normed in (True, False) if normed or w[8]])
def test_write(gpu, n, start, Hq, Hkv, D, bits, dims, trad, sections, turn, page, normed):
    """What lands in the pages and in the returned queries has the bits of
    apply_rotary on the same rows, whether a row comes alone or in a block."""
    rng = np.random.default_rng(sum(n) + D)
    T = sum(n)
    t = rotary_table(dims, base=1e6, traditional=trad, sections=sections, interleaved=turn)
    table, pages = tables(rng, [a + b for a, b in zip(start, n)], page)
    cache = PagedKVCache(pages, Hkv, D, page_size=page, bits=bits)
    off = i32([sum(n[:i]) for i in range(len(n) + 1)])
    q, k, v = rows(rng, T, Hq, D), rows(rng, T, Hkv, D), rows(rng, T, Hkv, D)
    norms = head_norms(weight(rng, D), weight(rng, D)) if normed else None
    given = t.axes > 1
    pos = some_positions(rng, t.axes, T) if given else np.concatenate([s + np.arange(m) for s, m in zip(start, n)])
    pos = torch.from_numpy(np.asarray(pos, np.int32)).cuda()
    qo = cache.write(k, v, table, i32(start), off, queries=q, rotary=t, norms=norms, positions=pos if given else None)
    cache.check_status()
    want_q, want_k = apply_rotary(t, q, k, pos, norms=norms)
    assert torch.equal(qo, want_q)
    plain = PagedKVCache(pages, Hkv, D, page_size=page, bits=bits)
    plain.write(want_k, v, table, i32(start), off)
    assert torch.equal(cache.k_pages, plain.k_pages) and torch.equal(cache.v_pages, plain.v_pages)
    if bits == 8:
        assert torch.equal(cache.k_scales, plain.k_scales)
    # positions other than the slots', with or without axes
    if not given and normed:
        moved = pos + 1000
        qm = cache.write(k, v, table, i32(start), off, queries=q, rotary=t, norms=norms, positions=moved)
        assert torch.equal(qm, apply_rotary(t, q, None, moved, norms=norms)[0])
        plain.write(apply_rotary(t, q, k, moved, norms=norms)[1], v, table, i32(start), off)
        assert torch.equal(cache.k_pages, plain.k_pages)
    # row by row: the same rows
    full = PagedKVCache(pages, Hkv, D, page_size=page, bits=bits)
    full.write(want_k, v, table, i32(start), off)
    alone = PagedKVCache(pages, Hkv, D, page_size=page, bits=bits)
    for b, (m, s) in enumerate(zip(n, start)):
        for i in range(min(m, 6)):
            at = sum(n[:b]) + i
            p1 = pos[..., at:at + 1].contiguous()
            one = alone.write(k[at:at + 1], v[at:at + 1], table[b:b + 1].contiguous(), i32([s + i]), rotary=t, norms=norms,
                              queries=q[at:at + 1], positions=p1)
            assert torch.equal(one[0], qo[at])
        got, want = stored(alone, table, b, s + min(m, 6)), stored(full, table, b, s + min(m, 6))
        assert all((g[:, s:] == w[:, s:]).all() for g, w in zip(got, want))


def test_write_without_queries_and_padded_rows(gpu):
    rng = np.random.default_rng(11)
    D, T = 64, 9
    t = rotary_table(D, base=1e4, sections=(12, 10, 10))
    table, pages = tables(rng, [10, 10], 32)
    cache = PagedKVCache(pages, 2, D, page_size=32)
    k, v, q = rows(rng, T, 2, D), rows(rng, T, 2, D), rows(rng, T, 4, D)
    norms = head_norms(None, weight(rng, D))
    pos = torch.from_numpy(some_positions(rng, 3, T)).cuda()
    off = i32([0, 3, 7])   # two rows belong to nobody
    assert cache.write(k, v, table, i32([2, 1]), off, rotary=t, norms=norms, positions=pos) is None
    first = cache.k_pages.clone()
    keep = torch.full((T, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = cache.write(k, v, table, i32([2, 1]), off, queries=q, rotary=t, norms=norms, positions=pos, out=keep)
    assert got is keep and torch.equal(cache.k_pages, first) and (keep[7:] == 7.0).all()
    want = apply_rotary(t, q, k, pos, norms=norms)
    assert torch.equal(keep[:7], want[0][:7])
    assert (stored(cache, table, 1, 5)[0][:, 1:] == num(want[1][3:7].transpose(0, 1))).all()


def test_captured_on_another_stream(gpu):
    rng = np.random.default_rng(12)
    D, T = 128, 6
    t = rotary_table(D, base=1e6, sections=(16, 24, 24))
    norms = head_norms(weight(rng, D), weight(rng, D))
    table, pages = tables(rng, [40, 40], 32)
    cache, other = (PagedKVCache(pages, 2, D, page_size=32, bits=8) for _ in range(2))
    q, k, v = rows(rng, T, 8, D), rows(rng, T, 2, D), rows(rng, T, 2, D)
    pos, start = torch.from_numpy(some_positions(rng, 3, T)).cuda(), i32([5, 30])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_rotary(t, q, k, pos, norms=norms)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a = apply_rotary(t, q, k, pos, norms=norms)
            b = cache.write(k, v, table, start, queries=q, rotary=t, norms=norms, positions=pos)
    torch.cuda.synchronize()
    for i in range(3):
        q.copy_(rows(rng, T, 8, D))
        k.copy_(rows(rng, T, 2, D))
        pos += 17
        want = apply_rotary(t, q, k, pos, norms=norms)
        other.write(k, v, table, start, queries=q, rotary=t, norms=norms, positions=pos)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1]) and torch.equal(b, want[0]), i
        assert torch.equal(cache.k_pages, other.k_pages) and torch.equal(cache.k_scales, other.k_scales), i


def test_refusals(gpu):
    t, t3 = rotary_table(64), rotary_table(64, sections=(8, 12, 12))
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    pos = i32([0, 1, 2, 3])
    w = torch.ones(64, device="cuda")
    for bad in (pos, pos.expand(2, 4), pos.expand(3, 4).t().contiguous()):
        with pytest.raises(ValueError):
            apply_rotary(t3, x, None, bad)
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos, norms=head_norms(torch.ones(32, device="cuda"), None))
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos, norms=head_norms(torch.ones(64), None))
    with pytest.raises(TypeError):
        apply_rotary(t, x, None, pos, norms=(w, w))
    cache = PagedKVCache(2, 2, 64)
    table, start = i32([[0]]), i32([0])
    with pytest.raises(ValueError):
        cache.write(x, x, table, start, norms=head_norms(w, w))
    with pytest.raises(ValueError):
        cache.write(x, x, table, start, positions=pos)
    with pytest.raises(ValueError):
        cache.write(x, x, table, start, rotary=t3)
    with pytest.raises(ValueError):
        cache.write(x, x, table, start, rotary=t, positions=pos[:3])
