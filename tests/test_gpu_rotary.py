"""GPU parity of the rotary positions with the float64 oracle.

Bound: one rounding to bf16 (2^-8 of the value) plus fp32's: cosine and sine
(2^-25 gain), the gain itself, the products and their sum (2^-24 of each) make
less than 2^-22 gain (|x1| + |x2|); the oracle's own angle at position 2^31 is
off by up to 2^-22, so 2^-21 in all.
"""

import math

import numpy as np
import pytest
import torch

from mtplx_amd.rotary import apply_rotary, rotary_table
from oracle import paged as O
from tests.paged_util import HALF, check_rows, i32, num, rows

pytestmark = pytest.mark.gpu


def _check(got, x, pos, t, what):
    want = O.rotate(num(x), pos, t.frequencies, t.dims, t.traditional, t.gain)
    a = np.abs(num(x))
    mate = a.copy()
    h = t.dims // 2
    i1, i2 = (np.arange(0, t.dims, 2), np.arange(1, t.dims, 2)) if t.traditional else (np.arange(h), np.arange(h) + h)
    mate[..., i1], mate[..., i2] = a[..., i2], a[..., i1]
    bound = HALF * np.abs(want) + abs(t.gain) * 2.0 ** -21 * (a + mate)
    bound[..., t.dims:] = 0.0
    check_rows(num(got), want, bound, what)


@pytest.mark.parametrize("T,Hq,Hkv,D,dims,trad", [
    (1, 40, 8, 128, 128, False), (1, 1, 1, 64, 64, True), (3, 5, 1, 64, 32, False), (17, 4, 2, 128, 96, True),
    (33, 2, 2, 256, 256, False), (100, 3, 1, 128, 24, False), (5, 3, 1, 80, 20, True), (7, 2, 1, 64, 2, False),
    (9, 2, 2, 40, 6, True), (513, 3, 1, 64, 64, False), (2500, 2, 1, 64, 48, True),
])
def test_matches_oracle(gpu, T, Hq, Hkv, D, dims, trad):
    rng = np.random.default_rng(T * 1000 + D + dims)
    t = rotary_table(dims, base=1e6, traditional=trad)
    q, k = rows(rng, T, Hq, D), rows(rng, T, Hkv, D)
    pos = rng.integers(0, 300000, T)
    qo, ko = apply_rotary(t, q, k, i32(pos))
    _check(qo, q, pos, t, "q")
    _check(ko, k, pos, t, "k")
    alone, none = apply_rotary(t, q, None, i32(pos))
    assert none is None and torch.equal(alone, qo)


@pytest.mark.parametrize("kw", [dict(scaling="yarn", factor=16.0, trained_positions=8192),
                                dict(scaling="ntk", factor=4.0), dict(scale=0.125), dict(gain=2.5)])
def test_scaled_and_far(gpu, kw):
    rng = np.random.default_rng(5)
    t = rotary_table(128, base=1e4, **kw)
    pos = np.array([0, 1, 8191, 1000003, 16777217, 2 ** 31 - 1, -1, -40000])
    q = rows(rng, len(pos), 2, 128)
    _check(apply_rotary(t, q, None, i32(pos.tolist()))[0], q, pos, t, str(kw))


def test_sine_and_cosine_of_every_turn(gpu):
    """Unit rows rotated by fractions all around: the outputs are the cosine
    and sine themselves, within bf16's rounding and fp32's of the angle's
    functions (2^-25, seen near their zeros, where bf16's is small)."""
    n = 1 << 16
    t = rotary_table(2, frequencies=[2 * math.pi / n * 1.0])
    x = torch.zeros((n, 1, 8), dtype=torch.bfloat16, device="cuda")
    x[..., 0] = 1.0
    pos = np.arange(n)
    y = num(apply_rotary(t, x, None, i32(pos))[0])[:, 0, :2]
    a = 2 * math.pi * pos / n
    want = np.stack([np.cos(a), np.sin(a)], -1)
    assert (np.abs(y - want) <= HALF * np.abs(want) + 2.0 ** -24).all()


def test_views_in_place_and_outputs(gpu):
    rng = np.random.default_rng(9)
    T, Hq, Hkv, D = 21, 4, 2, 64
    t = rotary_table(D, base=1e4)
    pos = i32(rng.integers(0, 5000, T))
    fused = rows(rng, T, (Hq + 2 * Hkv) * D)
    q = fused[:, :Hq * D].view(T, Hq, D)
    k = fused[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    want = apply_rotary(t, q.contiguous(), k.contiguous(), pos)
    got = apply_rotary(t, q, k, pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # rows that are not 16-byte aligned, and a transposed order
    odd = torch.empty(T * Hq * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, Hq, D)
    odd.copy_(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(apply_rotary(t, odd, k, pos)[0], want[0])
    assert torch.equal(apply_rotary(t, turned, k, pos)[0], want[0])
    # in place in the fused rows: V's columns stay
    keep = fused.clone()
    r = apply_rotary(t, q, k, pos, out=(q, k))
    assert r[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(fused[:, (Hq + Hkv) * D:], keep[:, (Hq + Hkv) * D:])
    # in place where halves are no whole chunks, and into a shifted view of the input
    t2 = rotary_table(24, base=1e4)
    x = rows(rng, T, Hq, D)
    want2 = apply_rotary(t2, x, None, pos)[0]
    y = x.clone()
    apply_rotary(t2, y, None, pos, out=(y, None))
    assert torch.equal(y, want2)
    buf = torch.cat([x, x[:1]])
    apply_rotary(t2, buf[:T], None, pos, out=(buf[1:], None))
    assert torch.equal(buf[1:], want2)


def test_refusals(gpu):
    t = rotary_table(64)
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    pos = i32([0, 1, 2, 3])
    with pytest.raises(TypeError):
        apply_rotary(t, x.float(), None, pos)
    with pytest.raises(ValueError):
        apply_rotary(t, x[0], None, pos)
    with pytest.raises(ValueError):
        apply_rotary(t, x, x[:3], pos)
    with pytest.raises(ValueError):
        apply_rotary(t, x, x[..., :32], pos)
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos[:3])
    with pytest.raises(ValueError):
        apply_rotary(t, x[..., :32].contiguous(), None, pos)
    with pytest.raises(ValueError):
        apply_rotary(rotary_table(64, device="cpu"), x, None, pos)
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos, out=(x[:2], None))
    with pytest.raises(ValueError):
        apply_rotary(t, x, x, pos, out=(x, x))
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos, out=(x[:1].expand(4, 2, 64), None))
    e = apply_rotary(t, x[:0], x[:0], pos[:0])
    assert e[0].shape == (0, 2, 64) and e[1].shape == (0, 2, 64)


def test_streams_and_graph(gpu):
    rng = np.random.default_rng(3)
    t = rotary_table(128, base=1e6)
    q, k = rows(rng, 64, 8, 128), rows(rng, 64, 2, 128)
    pos = i32(np.arange(64))
    want = apply_rotary(t, q, k, pos)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = apply_rotary(t, q, k, pos)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        cap = apply_rotary(t, q, k, pos)
    for step in range(3):
        pos.copy_(i32(np.arange(64) * (step + 2) + 5))
        q.copy_(rows(rng, 64, 8, 128))
        want = apply_rotary(t, q, k, pos)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap[0], want[0]) and torch.equal(cap[1], want[1])


def test_no_query_heads_refused(gpu):
    rng = np.random.default_rng(5)
    k = rows(rng, 4, 2, 128)
    with pytest.raises(ValueError):
        apply_rotary(rotary_table(128), k[:, :0], k, i32([0, 1, 2, 3]))
