"""Rotary positions on gfx950: pairs half a rotation apart or side by side,
the whole head or part of it, frequencies as trained or scaled for longer
contexts.

The reference rotates with ``mx.fast.rope`` (``dims``, ``traditional``, a base
and per-row offsets, ``tests/test_ragged_kv_cache.py:62-100``); here the
frequencies are a table made once (:func:`rotary_table`) and any packed
tokens are rotated at their own positions in one launch
(:func:`apply_rotary`). ``PagedKVCache.write`` takes the same table and
rotates on the way into the cache.

For pair i of position p, with angle ``a = p f_i``::

    y1 = gain (x1 cos a - x2 sin a)      y2 = gain (x1 sin a + x2 cos a)

in fp32, rounded once to bf16. Heads may be normalised on the way
(:func:`head_norms`), and a token may have several positions, each for its
own pairs (``sections``). The angle is reduced exactly (64-bit
fixed-point revolutions), so far positions are as precise as near ones.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field
from typing import Any, Sequence

import torch

from . import _lib

__all__ = ["HeadNorms", "RotaryTable", "apply_rotary", "head_norms", "rotary_table"]


@dataclass(frozen=True)
class RotaryTable:
    """Frequencies of ``dims / 2`` pairs: ``frequencies`` in radians per
    position (host, float64), ``phases`` the same as revolutions times 2^64
    (device, the bits of a uint64), ``gain`` the factor of the rotated values,
    ``axes`` how many positions a token has and ``axis`` (host) the one that
    each pair turns by (``axis_words``: as the kernels read it)."""

    dims: int
    traditional: bool
    gain: float
    frequencies: tuple
    phases: torch.Tensor
    axes: int = 1
    axis: tuple = ()
    axis_words: tuple = (0, 0, 0, 0)


@dataclass(frozen=True)
class HeadNorms:
    """RMS norms of each head of the queries and keys: fp32 weights ``[D]``
    (None: that side is not normalised) and the constant beside the mean."""

    queries: torch.Tensor | None
    keys: torch.Tensor | None
    eps: float
    args: Any = field(default=None, init=False, repr=False, compare=False)   # what every call with them passes

    def _take_args(self) -> None:
        object.__setattr__(self, "args", _lib.HeadArgs(_lib.ptr(self.queries), _lib.ptr(self.keys), axes=1, eps=self.eps))

    # A copy's calls pass the addresses of its own weights.
    def __getstate__(self):
        return {"queries": self.queries, "keys": self.keys, "eps": self.eps, "args": self.args is not None}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state, args=None)
        if state["args"]:
            self._take_args()


def head_norms(queries: torch.Tensor | None, keys: torch.Tensor | None, *, eps: float = 1e-6) -> HeadNorms:
    """:class:`HeadNorms` of weights ``[D]`` (any floating type; a copy in fp32
    is kept, so make it again after a change), for :func:`apply_rotary` and
    ``PagedKVCache.write``: ``w x / sqrt(mean(x^2) + eps)`` over each head, in
    fp32 (a head whose squares sum to 2^128 or more comes out as zeros)."""
    eps = float(eps)
    if not (math.isfinite(eps) and 0.0 <= eps < 3.0e38):
        raise ValueError(f"eps must be finite and not negative (got {eps})")
    if queries is None and keys is None:
        raise ValueError("give the queries' weight, the keys' or both")
    kept = []
    for name, w in (("queries", queries), ("keys", keys)):
        if w is not None:
            if not isinstance(w, torch.Tensor) or not w.is_floating_point() or w.dim() != 1:
                raise ValueError(f"the {name}' weight must be one dimension of floats")
            w = w.detach().to(torch.float32, copy=True).contiguous()
        kept.append(w)
    if None not in kept and (kept[0].shape != kept[1].shape or kept[0].device != kept[1].device):
        raise ValueError("the two weights must have one length and device")
    norms = HeadNorms(kept[0], kept[1], eps)
    norms._take_args()
    return norms


def rotary_frequencies(dims: int, *, base: float = 10000.0, scale: float = 1.0, scaling: str | None = None,
                       factor: float = 1.0, trained_positions: int = 0, fast_turns: float = 32.0,
                       slow_turns: float = 1.0) -> tuple[list[float], float]:
    """``(radians per position of each pair, gain)``.

    ``f_i = scale base^(-2 i / dims)``; ``scale`` below 1 squeezes positions
    evenly (``mx.fast.rope``'s ``scale``). ``scaling``:

    * ``"ntk"``: the base grows by ``factor^(dims / (dims - 2))``, so the
      slowest pair turns ``factor`` times slower and the fastest as before;
    * ``"yarn"``: pairs that make more than ``fast_turns`` turns over
      ``trained_positions`` stay, those below ``slow_turns`` turn ``factor``
      times slower, the pairs between are blended linearly in their index;
      the gain is ``0.1 ln(factor) + 1``.
    """
    if dims < 2 or dims % 2:
        raise ValueError(f"dims must be even and positive (got {dims})")
    for name, value in (("base", base), ("scale", scale), ("factor", factor)):
        if not (math.isfinite(value) and value > 0.0):
            raise ValueError(f"{name} must be positive and finite (got {value})")
    if scaling not in (None, "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'ntk' or 'yarn' (got {scaling!r})")
    if scaling is None and factor != 1.0:
        raise ValueError("factor belongs to a scaling ('ntk' or 'yarn'); use scale to squeeze positions evenly")
    if scaling == "ntk":
        if dims == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (dims / (dims - 2))
    freqs = [scale * base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling != "yarn":
        return freqs, 1.0
    if trained_positions < 1 or not fast_turns > slow_turns > 0.0 or base <= 1.0 or factor < 1.0:
        raise ValueError("yarn scaling needs trained_positions >= 1, fast_turns > slow_turns > 0, base > 1 and "
                         "factor >= 1")

    def pair_of(turns: float) -> float:   # index (in dims / 2 pairs) of the pair that makes so many turns
        return dims * math.log(scale * trained_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = max(math.floor(pair_of(fast_turns)), 0), min(math.ceil(pair_of(slow_turns)), dims - 1)
    for i, f in enumerate(freqs):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        freqs[i] = f * (1.0 - ramp) + f / factor * ramp
    return freqs, 0.1 * math.log(factor) + 1.0


MAX_AXES = 4


def _pair_axes(pairs: int, sections: Sequence[int], interleaved: bool) -> tuple:
    """The axis of each of ``pairs`` pairs."""
    counts = [int(n) for n in sections]
    A = len(counts)
    if not 1 <= A <= MAX_AXES or any(n < 1 for n in counts) or sum(counts) != pairs:
        raise ValueError(f"sections must be 1 to {MAX_AXES} positive counts of {pairs} pairs in all (got {counts})")
    if not interleaved:
        return tuple(a for a, n in enumerate(counts) for _ in range(n))
    if any(a + A * (n - 1) >= pairs for a, n in enumerate(counts) if a):
        raise ValueError(f"interleaved sections {counts}: an axis's last pair would lie past the {pairs} pairs")
    return tuple(i % A if i // A < counts[i % A] else 0 for i in range(pairs))


def rotary_table(dims: int, *, base: float = 10000.0, traditional: bool = False, scale: float = 1.0,
                 scaling: str | None = None, factor: float = 1.0, trained_positions: int = 0,
                 fast_turns: float = 32.0, slow_turns: float = 1.0, frequencies: Sequence[float] | None = None,
                 gain: float | None = None, sections: Sequence[int] | None = None, interleaved: bool = False,
                 device: Any = "cuda") -> RotaryTable:
    """The frequencies of :func:`rotary_frequencies`, or ``frequencies`` as
    given (radians per position, ``dims / 2`` of them, at most pi each), on
    ``device``. ``gain`` replaces the scaling's own.

    ``sections``: pairs that turn by each of several positions of a token (up
    to four axes: time, height and width of images and videos): the first
    ``sections[0]`` pairs by the first, and so on; ``interleaved``: pair i by
    axis ``i % axes`` while that axis has pairs left, else by the first."""
    if frequencies is None:
        freqs, own_gain = rotary_frequencies(dims, base=base, scale=scale, scaling=scaling, factor=factor,
                                             trained_positions=trained_positions, fast_turns=fast_turns,
                                             slow_turns=slow_turns)
    else:
        if dims < 2 or dims % 2:
            raise ValueError(f"dims must be even and positive (got {dims})")
        freqs, own_gain = [float(f) for f in frequencies], 1.0
        if len(freqs) != dims // 2:
            raise ValueError(f"expected {dims // 2} frequencies for dims={dims}, got {len(freqs)}")
    if dims > 256:
        raise ValueError(f"dims={dims} exceeds the largest head dim (256)")
    if not all(math.isfinite(f) and 0.0 <= f <= math.pi for f in freqs):
        raise ValueError("frequencies must lie in [0, pi] radians per position")
    gain = own_gain if gain is None else float(gain)
    if not math.isfinite(gain):
        raise ValueError("gain must be finite")
    # At most half a revolution each: the fixed-point value stays below 2^63.
    fixed = [min(round(f / (2.0 * math.pi) * 2.0 ** 64), 2 ** 63 - 1) for f in freqs]
    if sections is None and interleaved:
        raise ValueError("interleaved belongs to sections")
    axis = _pair_axes(dims // 2, sections, interleaved) if sections is not None else ()
    words = [0, 0, 0, 0]
    for i, a in enumerate(axis):   # two bits a pair
        words[i // 32] |= a << (2 * (i % 32))
    return RotaryTable(int(dims), bool(traditional), gain, tuple(freqs),
                       torch.tensor(fixed, dtype=torch.int64).to(device), len(sections) if axis else 1, axis,
                       tuple(w - (w >> 63 << 64) for w in words))   # (the bits, as signed)


def _positions(table: RotaryTable, positions: Any, T: int, device) -> torch.Tensor:
    """int32 ``[T]``, or ``[axes, T]`` of a table with sections, on ``device``."""
    if not (isinstance(positions, torch.Tensor) and positions.is_cuda):
        wide = torch.as_tensor(positions)
        positions = _int32("positions", wide, wide.device)
        if not torch.equal(positions.to(torch.int64), wide.to(torch.int64)):
            raise ValueError("positions must fit int32")
    pos = _int32("positions", positions, device, table.axes * T)
    if table.axes > 1 and tuple(pos.shape) != (table.axes, T):
        raise ValueError(f"positions must be [{table.axes}, {T}], a row for each axis (got {list(pos.shape)})")
    return pos


def _heads(table: RotaryTable, norms: HeadNorms | None, positions: torch.Tensor | None, D: int,
           device) -> _lib.HeadArgs:
    """The argument block of a call with head norms, several axes or positions
    of its own, its weights checked."""
    if norms is None:
        a = _lib.HeadArgs(axes=1)
    else:
        if not isinstance(norms, HeadNorms) or norms.args is None:
            raise TypeError(f"norms must come from head_norms (got {type(norms).__name__})")
        for name, w in (("queries", norms.queries), ("keys", norms.keys)):
            if w is not None:
                _on(device, f"norms.{name}", w)
                if w.shape[0] != D:
                    raise ValueError(f"norms.{name} has {w.shape[0]} weights, heads have {D} elements")
        a = _lib.HeadArgs.from_buffer_copy(norms.args)
    if positions is not None:
        a.positions = positions.data_ptr()
    if table.axes > 1:
        a.axes = table.axes
        a.axis0, a.axis1, a.axis2, a.axis3 = table.axis_words
    return a


def _rows(name: str, x: torch.Tensor, heads: int | None = None, dim: int | None = None):
    """``(x, tokens, heads, dim, token stride, head stride)`` of rows ``x``
    [T, H, D] bf16 on the GPU as the kernels read them: 16-byte aligned, strides
    of whole 16 bytes (other views are copied)."""
    if not x.is_cuda:
        raise RuntimeError(f"{name}: the paged operators run on the GPU only")
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16 (got {x.dtype})")
    shape = x.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or (dim is not None and shape[2] != dim):
        raise ValueError(f"{name} must be [tokens, {heads or 'heads'}, {dim or 'dim'}] (got {list(shape)})")
    T, H, D = shape
    t, h, d = x.stride()
    if d != 1 or t < 0 or t & 7 or h & 7 or h < D or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        t, h, d = x.stride()
        if T == 1 or H == 1:   # (a single row's stride is anything)
            t, h = H * D, D
            if D & 7:
                raise ValueError(f"{name}: a row of {D} elements is no whole 16 bytes")
    return x, T, H, D, t, h


def _writable(name: str, out: torch.Tensor, like: torch.Tensor):
    """``(out, token stride, head stride)`` of an output for the rows of ``like``:
    16-byte aligned rows that do not overlap, tokens or heads outermost."""
    if not isinstance(out, torch.Tensor):
        raise TypeError(f"{name} must be a tensor (got {type(out).__name__})")
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {list(like.shape)} {like.dtype} on {like.device}")
    T, H, D = out.shape
    t, h, d = out.stride()
    if H < 2:   # (a single one's stride is anything)
        h = D
    if T < 2:
        t = H * h
    apart = h >= D and t >= h * (H - 1) + D or t >= D and h >= t * (T - 1) + D
    if d != 1 or t & 7 or h & 7 or out.data_ptr() & 15 or not apart:
        raise ValueError(f"{name} must have 16-byte aligned rows that do not overlap")
    return out, t, h


_INT32 = (-2 ** 31, 2 ** 31 - 1)


def _int32(name: str, value: Any, device, numel: int | None = None) -> torch.Tensor:
    """``value`` as contiguous int32 on ``device``. What int32 cannot hold
    becomes the nearest that it can: no page of a pool and no position of a
    table (wrapped, it could be either)."""
    t = value if isinstance(value, torch.Tensor) else torch.as_tensor(value)
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        if t.numel() and (t.dtype is torch.bool or t.is_floating_point() or t.is_complex()):
            raise TypeError(f"{name} must hold integers (got {t.dtype})")
        if t.dtype in (torch.int64, torch.uint32, torch.uint64):
            top = t.dtype is torch.uint64
            t = t.to(device=device, dtype=torch.int64)
            if top:
                t = torch.where(t < 0, _INT32[1], t)   # (2^63 and on came out negative)
            t = t.clamp(*_INT32)
        t = t.to(device=device, dtype=torch.int32).contiguous()
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must hold {numel} values (got {t.numel()})")
    return t


def _on(device, name: str, t: torch.Tensor) -> None:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {device}")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device) -> int:
    """The current stream of ``device`` (as :func:`_lib.stream_handle`, without
    making a stream object where torch offers the handle itself)."""
    return _raw_stream(device.index) if _raw_stream is not None else _lib.stream_handle(device)


def _call(name: str, block: ctypes.Structure, device, more: ctypes.Structure | None = None) -> None:
    """Run an argument-block entry point, one of a single block or with ``more``,
    on ``device``'s current stream (the kernels of a call go to the current HIP
    device)."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            _call(name, block, device, more)
    elif more is None:
        _lib.call(name, ctypes.byref(block), _stream(device))
    else:
        _lib.call(name, ctypes.byref(block), ctypes.byref(more), _stream(device))


def _overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address spans of two views meet (two storages may hold the
    same memory, so storages are not compared)."""
    def span(x):
        lo = x.data_ptr()
        return lo, lo + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()

    if not (a.numel() and b.numel()):
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _apart(src: torch.Tensor, dst: torch.Tensor, in_place: bool = False) -> bool:
    """Whether a kernel may write the rows ``dst`` while it reads ``src``: they
    share no element (rows side by side do not) or, with ``in_place`` (an
    output and its own source), are the same view."""
    if not _overlaps(dst, src) or _interleaved(dst, src):
        return True
    return in_place and dst.data_ptr() == src.data_ptr() and dst.stride() == src.stride() and dst.shape == src.shape


def apply_rotary(table: RotaryTable, queries: torch.Tensor, keys: torch.Tensor | None, positions: Any, *,
                 norms: HeadNorms | None = None, out: tuple | None = None):
    """Rotate ``queries`` [T, Hq, D] and ``keys`` [T, Hkv, D] (or None) bf16 at
    ``positions`` [T], or [axes, T] of a table with sections (int32; may stay on
    the GPU, where a wider one counts as the nearest that fits). Returns
    ``(queries, keys)`` rotated, in new tensors or in ``out`` (a pair; the inputs
    themselves for in place). Views of a fused projection are read, and written,
    where they are.

    ``norms`` (:func:`head_norms`): each head is normalised first, all of it
    (elements that do not turn too), in the same pass and with one rounding."""
    q, T, Hq, D, qt, qh = _rows("queries", queries)
    device = q.device
    k, Hkv, kt, kh = None, 0, 0, 0
    if keys is not None:
        k, Tk, Hkv, _, kt, kh = _rows("keys", keys, None, D)
        if Tk != T:
            raise ValueError(f"queries have {T} tokens, keys {Tk}")
        _on(device, "keys", k)
    if Hq < 1:
        raise ValueError("queries have no heads")
    if D % 8 or D > 256 or table.dims > D:
        raise ValueError(f"head dim {D} must be a multiple of 8 up to 256 and hold the table's {table.dims} dims")
    pos = _positions(table, positions, T, device)
    _on(device, "table", table.phases)
    heads = None   # (the plain call pays for no part of it)
    if norms is not None or table.axes > 1:
        heads = _heads(table, norms, None if table.axes == 1 else pos, D, device)
    ko = None
    if out is None:
        qo = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=device)
        qot, qoh = Hq * D, D
        if k is not None:
            ko = torch.empty((T, Hkv, D), dtype=torch.bfloat16, device=device)
        kot, koh = Hkv * D, D
    else:
        qo, qot, qoh = _writable("out[0]", out[0], queries)
        kot = koh = 0
        if k is not None:
            ko, kot, koh = _writable("out[1]", out[1], keys)
        # An item of the kernel reads what it stores, unless the halves are no
        # whole chunks; tokens and heads go in no order.
        in_place = table.traditional or table.dims % 16 == 0
        if not _apart(q, qo, in_place) or (ko is not None and not _apart(q, ko)):
            q = q.clone(memory_format=torch.contiguous_format)
            qt, qh = Hq * D, D
        if k is not None and not (_apart(k, ko, in_place) and _apart(k, qo)):
            k = k.clone(memory_format=torch.contiguous_format)
            kt, kh = Hkv * D, D
        if ko is not None and _overlaps(qo, ko) and not _interleaved(qo, ko):
            raise ValueError("the two outputs overlap")
    if T == 0:
        return qo, ko
    if not Hkv:
        k = None
    block = _lib.RotaryArgs(
        q.data_ptr(), None if k is None else k.data_ptr(), qo.data_ptr(), None if k is None else ko.data_ptr(),
        pos.data_ptr(), table.phases.data_ptr(), T, Hq, Hkv, D, table.dims, table.traditional, table.gain, qt, qh, kt, kh,
        qot, qoh, kot, koh)
    if heads is None:
        _call("mtp_rotary", block, device)
    else:
        _call("mtp_rotary_heads", block, device, heads)
    return qo, ko


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views of one buffer of rows lie side by side in each row
    (the parts of a fused projection): equal token strides, disjoint columns."""
    if a.stride(0) != b.stride(0) or a.stride(0) <= 0:
        return False
    wide = a.stride(0) * a.element_size()
    (a0, an), (b0, bn) = ((x.data_ptr(), ((x.shape[1] - 1) * x.stride(1) + x.shape[2]) * x.element_size())
                          for x in (a, b))
    first, n, second = (a0, an, b0) if a0 <= b0 else (b0, bn, a0)
    gap = second - first
    return gap < wide and n <= gap and gap + (bn if first == a0 else an) <= wide
