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


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-5), dict(window=4, sinks=-1)])
def test_bad_scopes(kw):
    assert _run(_attn()[1], _lib.AttnScope(**kw)) == -1
    assert _lib.load().mtp_last_error().decode().startswith("mtp_paged_attn_scoped")


@pytest.mark.parametrize("bad", [dict(q=None), dict(ws=None), dict(ws_bytes=64), dict(Hq=3), dict(D=80), dict(scale=0.0)])
def test_bad_calls(bad):
    assert _run(_attn(**bad)[1], _lib.AttnScope(window=8, sinks=1)) < 0
    assert _lib.load().mtp_last_error().decode().startswith("mtp_paged_attn_scoped")


def test_null_blocks():
    assert _run(None, _lib.AttnScope(window=1)) == -1 and _run(_attn()[1], None) == -1
