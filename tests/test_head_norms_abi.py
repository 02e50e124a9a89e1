"""CPU checks of head norms and axes: argument block, refusals before any
launch, the axes of a table's pairs."""

import ctypes
import dataclasses

import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.rotary import HeadNorms, _heads, _pair_axes, head_norms, rotary_table
from oracle import paged as O
from tests.test_capi_symbols import HEADER, ROOT, _ctypes_fields, _struct_fields
from tests.test_paged_abi import _rotary, _write

CPU = torch.device("cpu")


def test_argument_block():
    want = _struct_fields(open(HEADER).read(), "mtp_head_args", typedef=True)
    assert [n for n, _ in want] == ["q_weight", "k_weight", "positions", "axis0", "axis1", "axis2", "axis3", "axes", "eps"]
    assert _struct_fields(open(f"{ROOT}/mtplx_amd/csrc/paged.hpp").read(), "mtp_head_args", typedef=False) == want
    assert _ctypes_fields(_lib.HeadArgs) == want


@pytest.mark.parametrize("kw", [dict(axes=0), dict(axes=5), dict(axes=3), dict(axes=1, eps=-1.0),
                                dict(axes=1, eps=float("nan")), dict(axes=1, eps=float("inf")), dict(axes=1, axis0=1),
                                dict(axes=3, positions=0x1000, axis0=3 << 62), dict(axes=2, positions=0x1000, axis0=-1)])
def test_refused_before_any_launch(kw):
    if "axis0" in kw:   # (as a signed word)
        kw = dict(kw, axis0=ctypes.c_longlong(kw["axis0"]).value)
    for name, block in (_rotary(), _write(dims=64, table=0x1000)):
        name += "_heads"
        assert getattr(_lib.load(), name)(ctypes.byref(block), ctypes.byref(_lib.HeadArgs(**kw)), None) == -1
        assert _lib.load().mtp_last_error().decode().startswith(name)


def test_refused_with_their_blocks():
    good = _lib.HeadArgs(axes=1)
    for name, block in (_rotary(q=None), _write(k=None, dims=64, table=0x1000), _write()):   # (the last: no rotation)
        assert getattr(_lib.load(), name + "_heads")(ctypes.byref(block), ctypes.byref(good), None) < 0
        assert getattr(_lib.load(), name + "_heads")(ctypes.byref(block), None, None) == -1
        assert getattr(_lib.load(), name + "_heads")(None, ctypes.byref(good), None) == -1


@pytest.mark.parametrize("pairs,sections,turn", [(64, (16, 24, 24), False), (64, (24, 20, 20), True), (32, (12, 10, 10), True),
                                                 (8, (8,), False), (8, (8,), True), (3, (1, 1, 1), True),
                                                 (128, (32, 32, 32, 32), True), (4, (3, 1), True)])
def test_axes_of_pairs(pairs, sections, turn):
    t = rotary_table(2 * pairs, sections=sections, interleaved=turn, device="cpu")
    assert t.axes == len(sections) and list(t.axis) == O.pair_axes(pairs, sections, turn).tolist()
    assert [t.axis.count(a) for a in range(t.axes)] == list(sections)
    pos = torch.zeros((t.axes, 1), dtype=torch.int32)
    a = _heads(t, None, pos, 2 * pairs, CPU)
    words = [w % 2 ** 64 for w in (a.axis0, a.axis1, a.axis2, a.axis3)]
    assert [words[i // 32] >> (2 * (i % 32)) & 3 for i in range(pairs)] == list(t.axis)


@pytest.mark.parametrize("sections,turn", [((), False), ((4, 3), False), ((8, 0), False), ((9, -1), False), ((2, 2, 2, 1, 1), False),
                                           ((1, 7), True), ((2, 5, 1), True)])
def test_bad_sections(sections, turn):
    with pytest.raises(ValueError):
        rotary_table(16, sections=sections, interleaved=turn, device="cpu")


def test_interleaved_needs_sections():
    with pytest.raises(ValueError):
        rotary_table(16, interleaved=True, device="cpu")
    assert _pair_axes(2, (1, 1), True) == (0, 1)


def test_norms_keep_a_copy():
    w = torch.ones(8, dtype=torch.float16)
    n = head_norms(w, w, eps=0.0)
    w.zero_()
    assert (n.queries == 1).all() and n.keys.dtype is torch.float32
    f = torch.ones(8)
    n = head_norms(None, f[::2])
    f.zero_()
    assert n.queries is None and (n.keys == 1).all() and n.keys.is_contiguous()
    for bad in (dict(queries=None, keys=None), dict(queries=torch.ones(2, 2), keys=None),
                dict(queries=torch.ones(4, dtype=torch.int32), keys=None), dict(queries=[1.0], keys=None),
                dict(queries=torch.ones(4), keys=torch.ones(5)), dict(queries=w, keys=None, eps=-1e-6),
                dict(queries=w, keys=None, eps=float("nan")), dict(queries=w, keys=None, eps=1e39)):
        with pytest.raises(ValueError):
            head_norms(**bad)


def test_norms_from_elsewhere_are_refused():
    """What a call passes holds the weights' addresses: others do not inherit it."""
    n = head_norms(torch.ones(8), None)
    t = rotary_table(8, device="cpu")
    assert _heads(t, n, None, 8, CPU).q_weight == n.queries.data_ptr()
    for other in (dataclasses.replace(n, eps=0.5), dataclasses.replace(n, queries=torch.ones(8)), HeadNorms(n.queries, None, 1e-6)):
        with pytest.raises(TypeError):
            _heads(t, other, None, 8, CPU)
