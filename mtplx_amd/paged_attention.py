"""Causal attention of new tokens over a paged KV cache on gfx950.

:func:`paged_sdpa` is to :class:`mtplx_amd.paged_kv_cache.PagedKVCache` what
``ragged_sdpa`` is to the padded cache (the reference's SDPA under
``ragged_causal_mask``, ``mtplx/ragged_attention.py:42``): the rule
``j <= q_start[b] + i`` applied implicitly. Requests of one call may bring one
token or thousands each: decode rows, verify rows, prompt chunks and whole
prompts run together.
"""

from __future__ import annotations

import math
from typing import Any

import torch

from . import _lib
from .paged_kv_cache import PagedKVCache
from .rotary import _call, _rows, _same_device, _writable, _overlaps

__all__ = ["paged_sdpa"]


def paged_sdpa(queries: torch.Tensor, cache: PagedKVCache, block_table: Any, q_start: Any, row_off: Any = None, *,
               max_rows: int | None = None, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` with grouped heads: ``queries`` [T, Hq, D] bf16
    (Hq 1 to 32 times the cache's kv heads) to ``[T, Hq, D]``.

    Request b's tokens are rows ``[row_off[b], row_off[b+1])`` (``row_off``
    None: ``T / B`` each) at positions ``q_start[b]`` on; token at position p
    sees positions 0..p of its request, which must be in the cache (write
    first, then attend). ``max_rows``: the longest request's rows, if known;
    calls of few rows then take the kernel for them (``row_off`` None: known).
    Rows past ``row_off[B]`` are not written, so they keep what ``out`` held
    (without ``out``: undefined). Rows that see no key are zeros;
    positions without a page count as absent and set ``cache.status()``.
    ``scale`` is positive; default ``1 / sqrt(D)``."""
    q = _rows("queries", queries, None, cache.head_dim)
    T, Hq, D = q.shape
    Hkv = cache.n_kv_heads
    if Hq % Hkv or not 1 <= Hq // Hkv <= 32:
        raise ValueError(f"query heads ({Hq}) must be 1 to 32 times the cache's kv heads ({Hkv})")
    table = cache._table(block_table)
    B = table.shape[0]
    start, off = cache._requests(T, B, q_start, row_off)
    _same_device(cache.device, queries=q)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite (got {scale})")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    else:
        out = _writable("out", out, queries)
        if _overlaps(out, q):
            q = q.clone(memory_format=torch.contiguous_format)
    if T == 0:
        return out
    rows = T // B if off is None else max(0, int(max_rows or 0))
    with torch.cuda.device(cache.device):
        nb = _lib.query("mtp_paged_attn_workspace_bytes", Hq, Hkv, D, rows)
    ws = _lib.WORKSPACES.get(nb, "paged_attn", cache.device)
    a = _lib.PagedAttnArgs(q=q.data_ptr(), out=out.data_ptr(), block_table=table.data_ptr(), q_start=start.data_ptr(),
                           row_off=_lib.ptr(off), ws=ws.data_ptr(), ws_bytes=ws.numel(), T=T, B=B,
                           width=table.shape[1], Hq=Hq, max_rows=rows, scale=scale, q_token=q.stride(0),
                           q_head=q.stride(1), out_token=out.stride(0), out_head=out.stride(1))
    cache._pages(a)
    _call("mtp_paged_attn", a, cache.device)
    return out
