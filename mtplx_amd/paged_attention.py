"""Causal attention of new tokens over a paged KV cache on gfx950.

:func:`paged_sdpa` is to :class:`mtplx_amd.paged_kv_cache.PagedKVCache` what
``ragged_sdpa`` is to the padded cache (the reference's SDPA under
``ragged_causal_mask``, ``mtplx/ragged_attention.py:42``): the rule
``j <= q_start[b] + i`` applied implicitly. Requests of one call may bring one
token or thousands each: decode rows, verify rows, prompt chunks and whole
prompts run together. A row may see a sliding window of its positions and the
first few (``window``, ``sinks``), and a batch whose requests share a long prefix
reads that once (``shared``).
"""

from __future__ import annotations

import math
import threading
from typing import Any

import torch

from . import _lib
from .attention_context import exact_verify_required
from .paged_kv_cache import PagedKVCache
from .rotary import _apart, _call, _on, _rows, _stream, _writable

__all__ = ["paged_sdpa"]


def paged_sdpa(queries: torch.Tensor, cache: PagedKVCache, block_table: Any, q_start: Any, row_off: Any = None, *,
               max_rows: int | None = None, scale: float | None = None, window: int | None = None, sinks: int = 0,
               shared: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` with grouped heads: ``queries`` [T, Hq, D] bf16
    (Hq 1 to 32 times the cache's kv heads) to ``[T, Hq, D]``.

    Request b's tokens are rows ``[row_off[b], row_off[b+1])`` (``row_off``
    None: ``T / B`` each) at positions ``q_start[b]`` on; token at position p
    sees positions 0..p of its request, which must be in the cache (write
    first, then attend). ``max_rows``: the longest request's rows, if known;
    calls of few rows then take the kernel for them (``row_off`` None: known).
    Rows past ``row_off[B]`` are not written, so they keep what ``out`` held
    (without ``out``: undefined). Rows that see no key are zeros; positions of
    the table without a page count as absent and set ``cache.status()``. A token
    at or past the table's end (``width * page_size``) sees the positions that the
    table has and sets nothing here: its ``write`` did.
    ``window``: a token at position p sees positions p - window + 1 to p alone
    (``window`` of them), and with ``sinks`` the first so many of its request
    too. What no new token sees is not read: the pages that hold nothing else may
    have been given back (-1 in the table).
    ``shared``: all requests that begin behind so many first positions hold the
    same keys there, in the same pages (their rows of ``block_table`` begin
    alike). A batch that shares a long prefix then reads it once instead of once
    for each request; the result is the same up to the order of sums. Requests
    that begin inside it, free slots among them, are as without. Not together
    with a window.
    ``scale`` is positive; default ``1 / sqrt(D)``. Refused inside
    ``exact_verify(True)``: how a row's sums are split depends on the lengths of
    the call's other requests."""
    if exact_verify_required():
        raise RuntimeError("paged_sdpa: a row's bits depend on the call's other requests, which a forward inside "
                           "exact_verify(True) must not (MTPLX_EXACT_T0_GUARD=0 disarms the guard)")
    q, T, Hq, D, qt, qh = _rows("queries", queries, None, cache.head_dim)
    Hkv = cache.n_kv_heads
    if Hq % Hkv or not 1 <= Hq // Hkv <= 32:
        raise ValueError(f"query heads ({Hq}) must be 1 to 32 times the cache's kv heads ({Hkv})")
    device = cache.device
    _on(device, "queries", q)
    table = cache._table(block_table)
    B, width = table.shape
    start, off = cache._requests(T, B, q_start, row_off)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite (got {scale})")
    scope = None
    if window is not None or sinks or shared:
        scope = _scope(window, sinks, int(shared), width * cache.page_size)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=device)
        ot, oh = Hq * D, D
    else:
        out, ot, oh = _writable("out", out, queries)
        if not _apart(q, out):
            q = q.clone(memory_format=torch.contiguous_format)
            qt, qh = Hq * D, D
    if T == 0:
        return out
    rows = T // B if off is None else 0 if max_rows is None else min(max(0, int(max_rows)), T)
    ws = _workspace(device, Hq, Hkv, D, rows) if scope is None else \
        _scoped_workspace(device, Hq, Hkv, D, rows, T, B, scope.shared)
    a = cache._block(_lib.PagedAttnArgs)
    a.q, a.out, a.block_table, a.q_start = q.data_ptr(), out.data_ptr(), table.data_ptr(), start.data_ptr()
    if off is not None:
        a.row_off = off.data_ptr()
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    a.T, a.B, a.width, a.Hq, a.max_rows, a.scale = T, B, width, Hq, rows, scale
    a.q_token, a.q_head, a.out_token, a.out_head = qt, qh, ot, oh
    with _LAUNCH:   # (its launches stay together: host threads may share a stream and so its workspace)
        if scope is None:
            _call("mtp_paged_attn", a, device)
        else:
            _call("mtp_paged_attn_scoped", a, device, scope)
    return out


def _scope(window: int | None, sinks: int, shared: int, covered: int) -> _lib.AttnScope | None:
    """What a row sees and what requests share, as an argument block (None: all
    up to itself, and nothing)."""
    window, sinks = None if window is None else int(window), int(sinks)
    if sinks < 0 or (window is not None and window < 1):
        raise ValueError(f"window must be positive and sinks not negative (got {window}, {sinks})")
    if sinks and window is None:
        raise ValueError("sinks belong to a window: without one every earlier token is visible")
    if not 0 <= shared <= covered:
        raise ValueError(f"shared must lie in the {covered} positions of the table (got {shared})")
    if shared and window is not None:
        raise ValueError("a window and shared positions do not go together")
    if shared:
        return _lib.AttnScope(0, 0, min(shared, 2 ** 31 - 1))
    # (no position of a table reaches 2^31: a longer window hides nothing)
    return None if window is None else _lib.AttnScope(min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1), 0)


_SPACES: dict = {}
_LAUNCH = threading.Lock()


def _workspace(device, Hq: int, Hkv: int, D: int, rows: int) -> torch.Tensor:
    """The partials' buffer of this device, stream and kind of call, looked up
    once (the pool keeps what it gave out allocated). A call that is being
    captured takes the graph's own memory: graphs captured on one stream may be
    replayed on two at once."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _workspace(device, Hq, Hkv, D, rows)
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(_lib.query("mtp_paged_attn_workspace_bytes", Hq, Hkv, D, rows), dtype=torch.uint8,
                           device=device)
    key = (device.index, _stream(device), Hq, Hkv, D, 0 < rows * (Hq // Hkv) <= 32)
    ws = _SPACES.get(key)
    if ws is None:
        nb = _lib.query("mtp_paged_attn_workspace_bytes", Hq, Hkv, D, rows)
        ws = _SPACES[key] = _lib.WORKSPACES.get(nb, "paged_attn", device)
    return ws


def _scoped_workspace(device, Hq: int, Hkv: int, D: int, rows: int, T: int, B: int, shared: int) -> torch.Tensor:
    """The same for a call with a window or a shared prefix, whose partials grow
    with its requests and rows."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _scoped_workspace(device, Hq, Hkv, D, rows, T, B, shared)
    def size() -> int:
        return _lib.query("mtp_paged_attn_scoped_workspace_bytes", Hq, Hkv, D, rows, T, B, shared)

    if torch.cuda.is_current_stream_capturing():
        return torch.empty(size(), dtype=torch.uint8, device=device)
    key = (device.index, _stream(device), Hq, Hkv, D, rows, B, shared and T, shared)
    ws = _SCOPED_SPACES.get(key)
    if ws is None:
        if len(_SCOPED_SPACES) >= 1024:   # (batches come in many shapes)
            _SCOPED_SPACES.clear()
        ws = _SCOPED_SPACES[key] = _lib.WORKSPACES.get(size(), "paged_attn_scoped", device)
    return ws


_SCOPED_SPACES: dict = {}
