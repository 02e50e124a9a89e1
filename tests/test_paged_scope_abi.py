"""CPU checks of attention over part of what a position sees: argument block and
what the entry point refuses before any launch."""

import ctypes

import pytest

from mtplx_amd import _lib
from tests.test_capi_symbols import HEADER, ROOT, _ctypes_fields, _struct_fields
from tests.test_paged_abi import _attn


def _run(block, scope):
    s = None if scope is None else ctypes.byref(scope)
    return _lib.load().mtp_paged_attn_scoped(None if block is None else ctypes.byref(block), s, None)


def test_argument_block():
    want = _struct_fields(open(HEADER).read(), "mtp_attn_scope", typedef=True)
    assert _struct_fields(open(f"{ROOT}/mtplx_amd/csrc/paged.hpp").read(), "mtp_attn_scope", typedef=False) == want
    assert _ctypes_fields(_lib.AttnScope) == want


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-5), dict(window=4, sinks=-1), dict(shared=-1),
                                dict(shared=32, window=4), dict(shared=32, sinks=4), dict(sinks=4),
                                dict(shared=193)])   # (the table covers 192)
def test_bad_scopes(kw):
    assert _run(_attn()[1], _lib.AttnScope(**kw)) == -1
    assert _lib.load().mtp_last_error().decode().startswith("mtp_paged_attn_scoped")


@pytest.mark.parametrize("bad", [dict(q=None), dict(ws=None), dict(ws_bytes=64), dict(Hq=3), dict(D=80), dict(scale=0.0),
                                 dict(B=1 << 20, row_off=0x1000), dict(width=(1 << 25) - 1)])
def test_bad_calls(bad):
    assert _run(_attn(**bad)[1], _lib.AttnScope(window=8, sinks=1)) < 0
    assert _lib.load().mtp_last_error().decode().startswith("mtp_paged_attn_scoped")


def test_workspace_bytes():
    plain = _lib.query("mtp_paged_attn_workspace_bytes", 40, 8, 128, 1)
    q = lambda *a: _lib.query("mtp_paged_attn_scoped_workspace_bytes", *a)  # noqa: E731
    assert q(40, 8, 128, 1, 16, 16, 8192) > q(40, 8, 128, 1, 16, 16, 0) > 0
    assert q(40, 8, 128, 1, 1, 1, 8192) == plain and q(3, 2, 128, 1, 16, 16, 8192) == 0   # nobody to share with
    assert q(40, 8, 128, 1, 2000, 2000, 0) == 2000 * 8 * 16                               # every head whole
    assert q(40, 8, 128, 1, 2000, 2000, 64) == plain                                      # too short to share
    block = _attn(T=4, B=2, width=100, ws_bytes=q(4, 2, 64, 2, 4, 2, 0))[1]
    assert _run(block, _lib.AttnScope(shared=6400)) == -3


def test_null_blocks():
    assert _run(None, _lib.AttnScope(window=1)) == -1 and _run(_attn()[1], None) == -1
