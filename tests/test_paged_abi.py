"""CPU checks of the paged operators: argument blocks, what the entry points
refuse before any launch, the frequencies of the rotary table, and the page
order against the verify step's own blocks."""

import ctypes
import math

import numpy as np
import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.paged_kv_cache import PagedKVCache
from mtplx_amd.rotary import apply_rotary, rotary_frequencies, rotary_table
from oracle import paged as O
from tests.test_capi_symbols import HEADER, ROOT, _ctypes_fields, _struct_fields


@pytest.mark.parametrize("name,cls", [("mtp_rotary_args", "RotaryArgs"), ("mtp_paged_write_args", "PagedWriteArgs"),
                                      ("mtp_paged_read_args", "PagedReadArgs"),
                                      ("mtp_paged_attn_args", "PagedAttnArgs")])
def test_argument_blocks(name, cls):
    want = _struct_fields(open(HEADER).read(), name, typedef=True)
    assert len(want) >= 15
    assert _struct_fields(open(f"{ROOT}/mtplx_amd/csrc/paged.hpp").read(), name, typedef=False) == want
    assert _ctypes_fields(getattr(_lib, cls)) == want


A = 0x1000   # an address that no refused call reads


def _rotary(**kw):
    a = dict(q=A, q_out=A, positions=A, table=A, T=4, Hq=2, D=64, dims=64, gain=1.0, q_token=128, q_head=64,
             qo_token=128, qo_head=64)
    return "mtp_rotary", _lib.RotaryArgs(**{**a, **kw})


def _write(**kw):
    a = dict(k=A, v=A, k_pages=A, v_pages=A, block_table=A, q_start=A, T=4, B=2, width=3, Hkv=2, D=64, page_size=64,
             num_pages=8, bits=16, k_token=128, k_head=64, v_token=128, v_head=64)
    return "mtp_paged_write", _lib.PagedWriteArgs(**{**a, **kw})


def _read(**kw):
    a = dict(k_pages=A, v_pages=A, block_table=A, k_out=A, v_out=A, B=2, width=3, count=5, Hkv=2, D=64, page_size=64,
             num_pages=8, bits=16)
    return "mtp_paged_read", _lib.PagedReadArgs(**{**a, **kw})


def _attn(**kw):
    a = dict(q=A, out=A, k_pages=A, v_pages=A, block_table=A, q_start=A, ws=A, ws_bytes=1 << 40, T=4, B=2, width=3,
             Hq=4, Hkv=2, D=64, page_size=64, num_pages=8, bits=16, scale=1.0, q_token=256, q_head=64, out_token=256,
             out_head=64)
    return "mtp_paged_attn", _lib.PagedAttnArgs(**{**a, **kw})


@pytest.mark.parametrize("call", [
    _rotary(q=None), _rotary(q_out=None), _rotary(positions=None), _rotary(T=0), _rotary(D=20), _rotary(D=264),
    _rotary(dims=65), _rotary(dims=66), _rotary(dims=-2), _rotary(table=None), _rotary(q=A + 8), _rotary(q_token=129),
    _rotary(q_head=32), _rotary(Hkv=1), _rotary(qo_token=-128),
    _write(k=None), _write(q_start=None), _write(D=96), _write(D=512), _write(page_size=48), _write(page_size=0),
    _write(num_pages=0), _write(width=0), _write(B=0), _write(T=0), _write(T=5), _write(bits=4), _write(bits=8),
    _write(k=A + 4), _write(v_token=12), _write(q=A), _write(dims=32), _write(dims=66, table=A),
    _write(width=1 << 26), _write(Hkv=0),
    _read(k_out=None), _read(count=-1), _read(bits=8), _read(D=32), _read(page_size=16), _read(v_out=A + 2),
    _attn(q=None), _attn(ws=None), _attn(ws_bytes=64), _attn(Hq=3), _attn(Hq=66), _attn(Hkv=0), _attn(T=3),
    _attn(scale=0.0), _attn(scale=-1.0), _attn(scale=float("nan")), _attn(scale=float("inf")), _attn(D=80),
    _attn(bits=8), _attn(q=A + 2), _attn(out_head=60), _attn(ws=A + 4),
])
def test_refused_before_any_launch(call):
    name, block = call
    lib = _lib.load()
    assert getattr(lib, name)(ctypes.byref(block), None) < 0
    assert lib.mtp_last_error().decode().startswith(name)
    with pytest.raises(_lib.MtpError, match=name):
        _lib.call(name, ctypes.byref(block), None)


def test_null_blocks():
    for name in ("mtp_rotary", "mtp_paged_write", "mtp_paged_read", "mtp_paged_attn"):
        assert getattr(_lib.load(), name)(None, None) == -1


def test_workspace_bytes():
    q = lambda *a: _lib.query("mtp_paged_attn_workspace_bytes", *a)  # noqa: E731
    assert q(40, 8, 128, 4) > 0 and q(40, 8, 128, 6) == q(40, 8, 128, 1)
    assert q(40, 8, 128, 7) > 3 * q(40, 8, 128, 6)      # 35 query rows per kv head: tiles of 256, not of 32
    assert q(40, 8, 128, 0) == q(40, 8, 128, 1000)
    assert q(3, 2, 128, 4) == 0


def test_cache_refusals():
    ok = dict(num_pages=2, n_kv_heads=1, head_dim=64, device="cpu")
    for bad in (dict(num_pages=0), dict(n_kv_heads=0), dict(head_dim=96), dict(page_size=16), dict(page_size=40),
                dict(bits=4)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**ok, **bad})
    c16, c8 = PagedKVCache(**ok), PagedKVCache(**ok, bits=8)
    assert c16.nbytes == 2 * 2 * 64 * 64 * 2 and c8.nbytes == 2 * 2 * 64 * (64 + 4)
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):   # no CPU fallback
        c16.write(x, x, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        apply_rotary(rotary_table(64, device="cpu"), x, None, torch.zeros(1, dtype=torch.int32))


def test_frequencies():
    f, gain = rotary_frequencies(8, base=10000.0)
    assert gain == 1.0 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-12)
    assert np.allclose(rotary_frequencies(8, scale=0.25)[0], np.array(f) / 4, rtol=1e-12)
    # ntk: the fastest pair as before, the slowest one factor times slower
    g, _ = rotary_frequencies(64, base=1e4, scaling="ntk", factor=8.0)
    plain, _ = rotary_frequencies(64, base=1e4)
    assert g[0] == plain[0] and np.isclose(g[-1], plain[-1] / 8.0, rtol=1e-12)
    # yarn: fast pairs as trained, slow ones factor times slower, monotone between
    y, gain = rotary_frequencies(128, base=1e6, scaling="yarn", factor=8.0, trained_positions=32768)
    plain, _ = rotary_frequencies(128, base=1e6)
    turns = np.array(plain) * 32768 / (2 * math.pi)
    ratio = np.array(y) / np.array(plain)
    assert np.allclose(ratio[turns > 40], 1.0) and np.allclose(ratio[turns < 0.8], 0.125)
    assert (np.diff(ratio) <= 1e-12).all() and math.isclose(gain, 0.1 * math.log(8.0) + 1.0)


@pytest.mark.parametrize("kw", [dict(dims=0), dict(dims=7), dict(dims=258), dict(dims=8, base=0.0),
                                dict(dims=8, base=float("inf")), dict(dims=8, scale=-1.0),
                                dict(dims=8, scaling="other"), dict(dims=8, factor=2.0),
                                dict(dims=2, scaling="ntk", factor=2.0), dict(dims=8, scaling="yarn", factor=2.0),
                                dict(dims=8, scaling="yarn", factor=0.5, trained_positions=4096),
                                dict(dims=8, frequencies=[1.0]), dict(dims=4, frequencies=[4.0, 1.0]),
                                dict(dims=4, frequencies=[float("nan"), 1.0]), dict(dims=4, gain=float("nan")),
                                dict(dims=4, base=1e-3)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        rotary_table(device="cpu", **kw)


def test_table_phases():
    t = rotary_table(4, frequencies=[math.pi, 0.25], gain=1.5, device="cpu")
    assert t.gain == 1.5 and t.phases.tolist() == [2 ** 63 - 1, round(0.25 / (2 * math.pi) * 2.0 ** 64)]
    # position * phase mod 2^64 is the turn's fraction, also far out and before 0
    for pos in (1, 1000003, 2 ** 31 - 1, -5):
        got = (pos * t.phases[1].item()) % 2 ** 64 / 2.0 ** 64
        want = (pos * 0.25 / (2 * math.pi)) % 1.0
        assert min(abs(got - want), 1 - abs(got - want)) < 2 ** 31 * 2.0 ** -52


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("kind", ["k", "v"])
def test_page_order_is_a_permutation(head_dim, bits, kind):
    at = O.page_order(kind, head_dim, bits)
    assert sorted(at.reshape(-1).tolist()) == list(range(32 * head_dim))
    if head_dim == 128 and bits == 16:
        from mtplx_amd.verify_step import kv_block_offsets
        assert at.reshape(-1).tolist() == kv_block_offsets(kind)


def test_quantised_rows():
    x = np.array([[0.0, 0.0], [1.0, -2.0], [2.0 ** -101, 0.0], [np.inf, 1.0], [1.0, np.nan]], np.float32)
    q, s = O.quantise_rows(x)
    assert q[1].tolist() == [64, -127] and s[1] == np.float32(2) / np.float32(127)   # 63.5 to even
    assert (q[[0, 2]] == 0).all() and (s[[0, 2]] == 0).all() and np.isnan(s[3:]).all()


def test_index_arrays_hold_integers():
    from mtplx_amd.rotary import _int32

    cpu = torch.device("cpu")
    assert _int32("positions", [3, 4], cpu).dtype is torch.int32 and _int32("positions", [], cpu).numel() == 0
    for bad in ([0.5], torch.ones(1), torch.ones(1, dtype=torch.bool)):
        with pytest.raises(TypeError):
            _int32("positions", bad, cpu)


def test_index_arrays_past_32_bits():
    """Entries that int32 cannot hold become the nearest it can, which is no page
    and no position of any cache; they never wrap to one that is."""
    from mtplx_amd.rotary import _int32

    cpu, top, low = torch.device("cpu"), 2 ** 31 - 1, -2 ** 31
    wide = [0, 5, -1, top, low, 2 ** 31, low - 1, 2 ** 32, 2 ** 32 + 3, -2 ** 32, 2 ** 63 - 1, -2 ** 63]
    want = [0, 5, -1, top, low, top, low, top, top, low, top, low]
    for value in (wide, torch.tensor(wide), torch.tensor(wide).view(2, 6).t()):
        got = _int32("block_table", value, cpu)
        assert got.dtype is torch.int32 and got.is_contiguous()
        assert got.tolist() == (want if got.dim() == 1 else torch.tensor(want).view(2, 6).t().tolist())
    assert _int32("block_table", torch.tensor([7, 2 ** 32 - 1], dtype=torch.uint32), cpu).tolist() == [7, top]
    assert _int32("block_table", torch.tensor([7, 255], dtype=torch.uint8), cpu).tolist() == [7, 255]
    big = torch.tensor([7, 2 ** 63 - 1, 2 ** 63 + 5, 2 ** 64 - 1], dtype=torch.uint64)
    assert _int32("block_table", big, cpu).tolist() == [7, top, top, top]
    same = torch.tensor([1, 2], dtype=torch.int32)
    assert _int32("block_table", same, cpu) is same


def test_yarn_counts_the_turns_that_scaled_positions_make():
    kw = dict(base=1e6, scaling="yarn", factor=8.0, trained_positions=32768)
    y, _ = rotary_frequencies(128, scale=0.125, **kw)
    plain, _ = rotary_frequencies(128, base=1e6, scale=0.125)
    turns = np.array(plain) * 32768 / (2 * math.pi)
    ratio = np.array(y) / np.array(plain)
    # one pair's step is a factor of 1e6^(1/64) = 1.24: whole pairs to either side of 32 and 1 turns
    assert np.allclose(ratio[turns > 40], 1.0) and np.allclose(ratio[turns < 0.8], 0.125)
    assert (ratio[(turns < 25) & (turns > 1.3)] < 1.0).all() and (ratio[(turns < 25) & (turns > 1.3)] > 0.125).all()
