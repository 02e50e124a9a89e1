"""A paged KV cache on gfx950, in 16 or 8 bits.

The reference's ragged cache (``mtplx/ragged_kv_cache.py:71``,
:class:`mtplx_amd.ragged_kv_cache.RaggedBatchKVCache` here) holds one padded
buffer for a batch. This one holds a pool of pages; a request's keys are in
the pages that its row of a block table names, so requests of any length come
and go without copies and may share the pages of a common prefix. Which page
belongs to whom is the caller's: the cache stores, it does not allocate.

Pages lie in the order in which :func:`mtplx_amd.paged_attention.paged_sdpa`
loads them (``include/mtplx_amd.h``); :meth:`PagedKVCache.read` gives rows
back in the reference's ``[B, Hkv, count, D]``.

With ``bits=8`` each token's row of each head is stored as int8 and one fp32
scale (``scale = max|x| / 127``, values rounded to nearest even): 0.52 of the
bytes at head dim 128. The largest error of a value is half a step,
``max|x| / 254``.
"""

from __future__ import annotations

from typing import Any

import torch

from . import _lib
from .rotary import RotaryTable, _apart, _call, _int32, _on, _rows, _writable

__all__ = ["PagedKVCache"]


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` keys for ``n_kv_heads`` heads."""

    def __init__(self, num_pages: int, n_kv_heads: int, head_dim: int, *, page_size: int = 64, bits: int = 16,
                 device: Any = "cuda") -> None:
        if num_pages < 1 or n_kv_heads < 1:
            raise ValueError(f"need at least one page and one kv head (got {num_pages}, {n_kv_heads})")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256 (got {head_dim})")
        if page_size < 32 or page_size % 32:
            raise ValueError(f"page_size must be a positive multiple of 32 (got {page_size})")
        if bits not in (8, 16):
            raise ValueError(f"bits must be 8 or 16 (got {bits})")
        self.num_pages, self.n_kv_heads, self.head_dim = int(num_pages), int(n_kv_heads), int(head_dim)
        self.page_size, self.bits = int(page_size), int(bits)
        shape = (self.num_pages, self.n_kv_heads, self.page_size // 32, 32 * self.head_dim)
        dtype = torch.int8 if bits == 8 else torch.bfloat16
        self._k = torch.zeros(shape, dtype=dtype, device=device)
        self._v = torch.zeros_like(self._k)
        self._ks = self._vs = None
        if bits == 8:
            self._ks = torch.zeros(shape[:2] + (self.page_size,), dtype=torch.float32, device=device)
            self._vs = torch.zeros_like(self._ks)
        self._status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device = self._k.device
        # What every call over this cache passes, filled in once.
        held = dict(k_pages=self._k.data_ptr(), v_pages=self._v.data_ptr(), k_scales=_lib.ptr(self._ks),
                    v_scales=_lib.ptr(self._vs), status=self._status.data_ptr(), Hkv=self.n_kv_heads, D=self.head_dim,
                    page_size=self.page_size, num_pages=self.num_pages, bits=self.bits)
        self._blocks = {cls: cls(**held) for cls in (_lib.PagedWriteArgs, _lib.PagedReadArgs, _lib.PagedAttnArgs)}

    # The pool's tensors (their contents may be copied in and out; the cache
    # keeps the tensors themselves).
    @property
    def k_pages(self) -> torch.Tensor:
        return self._k

    @property
    def v_pages(self) -> torch.Tensor:
        return self._v

    @property
    def k_scales(self) -> torch.Tensor | None:
        return self._ks

    @property
    def v_scales(self) -> torch.Tensor | None:
        return self._vs

    @property
    def nbytes(self) -> int:
        held = (self._k, self._v, self._ks, self._vs)
        return sum(t.numel() * t.element_size() for t in held if t is not None)

    def status(self) -> torch.Tensor:
        """Device status word (int32 [1]): nonzero once a call met a position
        that the block table has no page for (its row was skipped)."""
        return self._status

    def check_status(self) -> None:
        """Raise :class:`MtpError` if a call since the last check met a position
        without a page. Waits for the device, so calls on every stream count;
        one that another host thread makes meanwhile may go unseen."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        if int(self._status.item()) != 0:
            self._status.zero_()
            raise _lib.MtpError("paged_kv_cache", -1, "a position without a page of the pool (status word set)")

    # -- shared by the calls over this cache --------------------------------------
    def _block(self, cls):
        return cls.from_buffer_copy(self._blocks[cls])

    def _table(self, block_table: Any) -> torch.Tensor:
        t = _int32("block_table", block_table, self.device)
        if t.dim() != 2 or t.shape[0] < 1 or t.shape[1] < 1:
            raise ValueError(f"block_table must be [requests, pages] (got {list(t.shape)})")
        if t.shape[1] * self.page_size > 0x7fffffff:
            raise ValueError("block_table covers more than 2^31 - 1 positions")
        return t

    def _requests(self, tokens: int, B: int, q_start: Any, row_off: Any):
        start = _int32("q_start", q_start, self.device, B)
        if row_off is None:
            if tokens % B:
                raise ValueError(f"{tokens} tokens are no whole rows of {B} requests: give row_off")
            return start, None
        return start, _int32("row_off", row_off, self.device, B + 1)

    # -- writes and reads ------------------------------------------------------------
    def write(self, keys: torch.Tensor, values: torch.Tensor, block_table: Any, q_start: Any, row_off: Any = None, *,
              max_rows: int | None = None, queries: torch.Tensor | None = None, rotary: RotaryTable | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Store the new tokens' ``keys`` / ``values`` [T, Hkv, D] bf16.

        Request b's tokens are rows ``[row_off[b], row_off[b+1])`` (``row_off``
        None: ``T / B`` each) at positions ``q_start[b]`` on, in the pages of
        ``block_table[b]`` (int32 ``[B, pages]``, -1 where there is none). All
        three may stay on the GPU. Rows past ``row_off[B]`` belong to nobody: they
        are not stored, nor written in the returned tensor (undefined there).
        ``max_rows``: the longest request's rows, if the caller knows (a hint
        that sizes the launch). With ``rotary`` keys are rotated at their
        positions on the way, and ``queries`` [T, Hq, D] into the returned
        tensor (or ``out``), as :func:`apply_rotary` would. Without ``rotary``
        ``queries`` has no meaning and is refused.

        Two tokens of one call must not share a slot. A position without a
        page is skipped and sets :meth:`status`."""
        D, H = self.head_dim, self.n_kv_heads
        k, T, _, _, kt, kh = _rows("keys", keys, H, D)
        v, Tv, _, _, vt, vh = _rows("values", values, H, D)
        if Tv != T:
            raise ValueError(f"keys have {T} tokens, values {Tv}")
        device = self.device
        _on(device, "keys", k)
        _on(device, "values", v)
        if queries is not None and rotary is None:
            raise ValueError("queries are taken to be rotated: give rotary with them")
        if rotary is not None:
            if rotary.dims > D:
                raise ValueError(f"the rotary table's {rotary.dims} dims exceed the head dim {D}")
            _on(device, "rotary", rotary.phases)
        table = self._table(block_table)
        B, width = table.shape
        start, off = self._requests(T, B, q_start, row_off)
        q = qo = None
        if queries is not None:
            q, Tq, Hq, _, qt, qh = _rows("queries", queries, None, D)
            if Tq != T:
                raise ValueError(f"keys have {T} tokens, queries {Tq}")
            _on(device, "queries", q)
            if out is None:
                qo = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=device)
                qot, qoh = Hq * D, D
            else:
                qo, qot, qoh = _writable("out", out, queries)
                for name, x in (("keys", k), ("values", v)):
                    if not _apart(x, qo):
                        raise ValueError(f"out overlaps {name}")
                if not _apart(q, qo, rotary.traditional or rotary.dims % 16 == 0):
                    q = q.clone(memory_format=torch.contiguous_format)
                    qt, qh = Hq * D, D
        if T == 0:
            return qo
        a = self._block(_lib.PagedWriteArgs)
        a.k, a.v, a.k_token, a.k_head, a.v_token, a.v_head = k.data_ptr(), v.data_ptr(), kt, kh, vt, vh
        a.block_table, a.q_start, a.T, a.B, a.width = table.data_ptr(), start.data_ptr(), T, B, width
        if off is not None:
            a.row_off = off.data_ptr()
            if max_rows is not None and max_rows > 0:
                a.max_rows = min(int(max_rows), T)
        if rotary is not None:
            a.table, a.dims, a.gain = rotary.phases.data_ptr(), rotary.dims, rotary.gain
            a.traditional = rotary.traditional
        if q is not None and Hq:
            a.q, a.q_out, a.Hq = q.data_ptr(), qo.data_ptr(), Hq
            a.q_token, a.q_head, a.qo_token, a.qo_head = qt, qh, qot, qoh
        _call("mtp_paged_write", a, device)
        return qo

    def read(self, block_table: Any, count: int, *, start: Any = None, lengths: Any = None):
        """``(keys, values)`` bf16 ``[B, Hkv, count, D]`` of positions
        ``start[b]`` (None: 0) on. Positions at or past ``lengths[b]`` (None:
        all are live) read as zeros and touch no page; live positions without a
        page read as zeros and set :meth:`status`."""
        table = self._table(block_table)
        B, count = table.shape[0], int(count)
        if count < 0:
            raise ValueError(f"count must not be negative (got {count})")
        first = None if start is None else _int32("start", start, self.device, B)
        ends = None if lengths is None else _int32("lengths", lengths, self.device, B)
        shape = (B, self.n_kv_heads, count, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        if count:
            a = self._block(_lib.PagedReadArgs)
            a.block_table, a.k_out, a.v_out = table.data_ptr(), k.data_ptr(), v.data_ptr()
            a.start, a.lengths = _lib.ptr(first), _lib.ptr(ends)
            a.B, a.width, a.count = B, table.shape[1], count
            _call("mtp_paged_read", a, self.device)
        return k, v
