"""GPU parity of the paged cache's writes and reads: stored bits against the
oracle's quantisation and page order, exact."""

import numpy as np
import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import apply_rotary, rotary_table
from oracle import paged as O
from tests.paged_util import i32, num, rows, stored, tables

pytestmark = pytest.mark.gpu


def _expect(x, bits):
    """float64 values that bf16 rows [.., D] stand for once they are stored."""
    if bits == 16:
        return num(x)
    q, s = O.quantise_rows(x.float().cpu().numpy())
    return q.astype(np.float64) * s.astype(np.float64)[..., None]


def _as_read(values, bits):
    """What a read of stored values gives (8 bits: one rounding of q * scale in
    fp32, then one to bf16)."""
    if bits == 16:
        return values
    return torch.from_numpy(values.astype(np.float32)).to(torch.bfloat16).double().numpy()


CASES = [  # (new tokens, first position) of each request; head dim, kv heads, page, bits
    ([1], [0], 128, 8, 64, 16), ([1], [63], 128, 1, 64, 8), ([1, 1, 1], [31, 32, 100], 64, 2, 32, 8),
    ([40, 0, 7, 1], [0, 5, 30, 95], 128, 2, 64, 16), ([40, 0, 7, 1], [0, 5, 30, 95], 128, 2, 64, 8),
    ([33], [31], 256, 1, 32, 16), ([97, 64], [1, 64], 64, 3, 96, 8), ([200, 3], [17, 500], 256, 2, 256, 8),
    ([5] * 70, list(range(70)), 64, 1, 32, 16), ([1] * 130, list(range(0, 1300, 10)), 128, 1, 128, 8),
]


@pytest.mark.parametrize("n,start,D,H,page,bits", CASES)
@pytest.mark.parametrize("turn", [False, True])
def test_write_and_read(gpu, n, start, D, H, page, bits, turn):
    rng = np.random.default_rng(sum(n) * 7 + D + bits + turn)
    T, B = sum(n), len(n)
    table, pages = tables(rng, [s + m for s, m in zip(start, n)], page)
    c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
    # what was there before: must survive beside the new rows
    old = rows(rng, pages * page, H, D)
    every = torch.arange(pages, dtype=torch.int32, device="cuda").unsqueeze(1)
    c.write(old, old * 2, every, torch.zeros(pages, dtype=torch.int32, device="cuda"))
    before = [stored(c, table, b, -(-(start[b] + n[b]) // page) * page) for b in range(B)]
    want_old = _expect(old, bits).reshape(pages, page, H, D)
    for b in range(B):
        ids = table[b][table[b] >= 0].long().cpu().numpy()[:-(-(start[b] + n[b]) // page)]
        assert np.array_equal(before[b][0], want_old[ids].reshape(-1, H, D).transpose(1, 0, 2))
    k, v, q = rows(rng, T + 3, H, D), rows(rng, T + 3, H, D), rows(rng, T + 3, 3 * H, D)
    off = i32(np.concatenate([[0], np.cumsum(n)]))
    out = torch.full_like(q, 7.0)
    rot = rotary_table(D, base=1e4) if turn else None
    got = c.write(k, v, table, i32(start), off, max_rows=max(n), queries=q if turn else None, rotary=rot,
                  out=out if turn else None)
    pos = np.concatenate([np.arange(s, s + m) for s, m in zip(start, n)])
    if turn:   # the same bits as the rotation by itself; rows of nobody stay
        wq, k = apply_rotary(rot, q[:T], k[:T], i32(pos))
        assert got is out and torch.equal(out[:T], wq) and (out[T:] == 7.0).all()
    else:
        assert got is None
    kw, vw = _expect(k[:T], bits), _expect(v[:T], bits)
    for b in range(B):
        lo, s, e = int(off[b]), start[b], start[b] + n[b]
        after = stored(c, table, b, -(-e // page) * page)
        for x, was, new in ((after[0], before[b][0], kw), (after[1], before[b][1], vw)):
            assert np.array_equal(x[:, s:e], new[lo:lo + n[b]].transpose(1, 0, 2))
            assert np.array_equal(x[:, :s], was[:, :s]) and np.array_equal(x[:, e:], was[:, e:])
    assert int(c.status().item()) == 0
    # back: from the first new position, the requests' own lengths
    count = max(n) + 2
    ends = i32([s + m for s, m in zip(start, n)])
    kr, vr = (num(x) for x in c.read(table, count, start=i32(start), lengths=ends))
    for b in range(B):
        lo = int(off[b])
        for x, new in ((kr[b], kw), (vr[b], vw)):
            assert np.array_equal(x[:, :n[b]], _as_read(new[lo:lo + n[b]].transpose(1, 0, 2), bits))
            assert (x[:, n[b]:] == 0).all()
    whole = c.read(table, page)   # a first page, of requests that have one
    for b in range(B):
        if start[b] + n[b] >= page:
            assert np.array_equal(num(whole[0][b]), _as_read(stored(c, table, b, page)[0], bits))
    assert int(c.status().item()) == (0 if (table[:, 0] >= 0).all() else 1)


@pytest.mark.parametrize("bits", [8, 16])
def test_uniform_rows_and_views(gpu, bits):
    """row_off None, K and V as views of one fused projection, int64 tables."""
    rng = np.random.default_rng(4)
    B, L, H, D, page = 3, 5, 2, 64, 32
    start = [30, 0, 61]
    table, pages = tables(rng, [s + L for s in start], page)
    fused = rows(rng, B * L, 4 * H * D)
    k, v = (fused[:, i * H * D:(i + 1) * H * D].view(B * L, H, D) for i in (2, 3))
    a, b = (PagedKVCache(pages, H, D, page_size=page, bits=bits) for _ in range(2))
    a.write(k, v, table.long(), torch.tensor(start))
    b.write(k.contiguous(), v.contiguous(), table, i32(start), i32([0, 5, 10, 15]))
    for x, y in zip(a.read(table, 70, lengths=i32([35, 5, 66])), b.read(table, 70, lengths=i32([35, 5, 66]))):
        assert torch.equal(x, y)
    assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)
    assert int(a.status().item()) == 0


@pytest.mark.parametrize("bits", [8, 16])
def test_positions_without_a_page(gpu, bits):
    rng = np.random.default_rng(6)
    H, D, page = 1, 128, 32
    c = PagedKVCache(4, H, D, page_size=page, bits=bits)
    table = i32([[0, -1], [2, 9], [3, 1]])   # 9: outside the pool
    k, v = rows(rng, 3 * 40, H, D), rows(rng, 3 * 40, H, D)
    c.write(k, v, table, i32([0, 10, 40]))   # request 2 runs past its 64 positions
    with pytest.raises(_lib.MtpError):
        c.check_status()
    c.check_status()   # cleared
    kr, _ = c.read(table, 64)
    with pytest.raises(_lib.MtpError):
        c.check_status()
    kw = _as_read(_expect(k, bits), bits)[:, 0].reshape(3, 40, D)
    got = num(kr)[:, 0]
    assert np.array_equal(got[0, :32], kw[0, :32]) and (got[0, 32:] == 0).all()
    assert (got[1, :10] == 0).all() and np.array_equal(got[1, 10:32], kw[1, :22]) and (got[1, 32:] == 0).all()
    assert np.array_equal(got[2, 40:], kw[2, :24]) and (got[2, :40] == 0).all()
    # positions past a length touch no page, live ones before 0 or past the table have none
    c.read(table, 64, lengths=i32([32, 32, 64]))
    c.check_status()
    assert (num(c.read(table, 8, start=i32([-20, -8, 64]))[0]) == 0).all()
    with pytest.raises(_lib.MtpError):
        c.check_status()
    # a first position far outside any table
    c.write(k[:3], v[:3], table, i32([2 ** 31 - 1, -2 ** 31, 2 ** 30]))
    with pytest.raises(_lib.MtpError):
        c.check_status()
    assert torch.equal(c.read(table, 64)[0], kr)


def test_row_offsets_are_clamped(gpu):
    """Offsets outside the packed rows, or falling, name no row outside them."""
    rng = np.random.default_rng(8)
    c = PagedKVCache(4, 1, 64, page_size=32)
    k = rows(rng, 6, 1, 64)
    table = i32([[0], [1], [2], [3]])
    c.write(k, k, table, i32([0, 0, 0, 0]), i32([-5, 2, 1, 4, 99]))
    got = num(c.read(table, 8)[0])[:, 0]
    kn = num(k)[:, 0]
    for b, (lo, hi) in enumerate([(0, 2), (2, 2), (1, 4), (4, 6)]):
        assert np.array_equal(got[b, :hi - lo], kn[lo:hi]) and (got[b, hi - lo:] == 0).all()


def test_rows_that_are_not_numbers(gpu):
    """8 bits: NaN or an infinity makes its own row read as NaN and no other;
    tiny rows are zeros, huge ones keep their scale."""
    x = torch.ones((6, 1, 64), dtype=torch.bfloat16, device="cuda")
    x[1, 0, 5] = float("nan")
    x[2, 0, 9] = float("inf")
    x[3] = 2.0 ** -110
    x[4, 0, 0] = 3.0e38
    x[5] = 0.0
    c = PagedKVCache(1, 1, 64, page_size=32, bits=8)
    c.write(x, x, i32([[0]]), i32([0]))
    k, v = c.read(i32([[0]]), 6)
    for got in (num(k)[0, 0], num(v)[0, 0]):
        assert (got[0] == 1).all() and np.isnan(got[1:3]).all() and (got[[3, 5]] == 0).all()
        assert abs(got[4, 0] / 3.0e38 - 1) < 0.01 and (got[4, 1:] == 0).all()


def test_pages_past_32_bit_offsets(gpu):
    """The last page of a pool of more than 2^31 elements."""
    D, H, page = 256, 8, 256
    pages = 2 ** 31 // (D * H * page) + 3
    rng = np.random.default_rng(1)
    for bits in (16, 8):
        c = PagedKVCache(pages, H, D, page_size=page, bits=bits)
        table = i32([[pages - 1]])
        k, v = rows(rng, 40, H, D), rows(rng, 40, H, D)
        c.write(k, v, table, i32([7]))
        for got, x in zip(c.read(table, 40, start=i32([7])), (k, v)):
            assert np.array_equal(num(got)[0], _as_read(_expect(x, bits).transpose(1, 0, 2), bits))
        assert not c.k_pages[:pages - 1].any().item() and not c.v_pages[:pages - 1].any().item()
        del c


def test_refusals(gpu):
    c = PagedKVCache(2, 2, 64, page_size=32)
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    table, start, rot = i32([[0], [1]]), i32([0, 0]), rotary_table(64)
    bad = [lambda: c.write(x, x[:3], table, start), lambda: c.write(x[:, :1], x[:, :1], table, start),
           lambda: c.write(x[:3], x[:3], table, start), lambda: c.write(x, x, table[0], start),
           lambda: c.write(x, x, table, start[:1]), lambda: c.write(x, x, table, start, i32([0, 4])),
           lambda: c.write(x, x, table, start, queries=q), lambda: c.write(x, x, table, start, queries=q[:2], rotary=rot),
           lambda: c.write(x, x, table, start, rotary=rotary_table(128)),
           lambda: c.write(x, x, table, start, rotary=rotary_table(64, device="cpu")),
           lambda: c.write(x, x, table, start, queries=q, rotary=rot, out=q[:, :2]),
           lambda: c.write(x, x, table, start, queries=x, rotary=rot, out=x),
           lambda: c.read(table, -1), lambda: c.read(table, 4, start=start[:1]),
           lambda: c.read(table, 4, lengths=i32([1, 2, 3]))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        c.write(x.float(), x.float(), table, start)
    assert c.write(x[:0], x[:0], table, start) is None
    assert c.read(table, 0)[0].shape == (2, 2, 0, 64)
    assert not c.k_pages.any().item()


def test_graph_replays_follow_their_inputs(gpu):
    rng = np.random.default_rng(12)
    B, H, D, page = 4, 2, 128, 64
    table, pages = tables(rng, [256] * B, page)
    rot = rotary_table(D, base=1e5)
    caches = [PagedKVCache(pages, H, D, page_size=page, bits=8) for _ in range(2)]
    k, v, q = rows(rng, 10, H, D), rows(rng, 10, H, D), rows(rng, 10, 6, D)
    off, start = i32([0, 1, 4, 4, 9]), i32([0, 50, 9, 100])
    step = lambda c: (c.write(k, v, table, start, off, queries=q, rotary=rot),  # noqa: E731
                      *c.read(table, 5, start=start, lengths=start + off[1:] - off[:-1]))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step(caches[0])
    for i in range(3):
        k.copy_(rows(rng, 10, H, D))
        start.copy_(i32([i, 50 + 20 * i, 9, 100 + 31 * i]))
        off.copy_(i32([0, 2 + i, 4, 4, 8 + i]))
        want = step(caches[1])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0][:8 + i], want[0][:8 + i])   # rows of nobody are undefined
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert torch.equal(caches[0].k_pages, caches[1].k_pages) and torch.equal(caches[0].v_scales, caches[1].v_scales)
