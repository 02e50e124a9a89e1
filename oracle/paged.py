"""Float64 NumPy restatement of the paged path: rotary positions, the 8-bit
rows of the cache, the order of a page, and causal attention with grouped
heads over the keys that each position sees."""

from __future__ import annotations

import math

import numpy as np


def rotate(x: np.ndarray, positions, frequencies, dims: int, traditional: bool, gain: float = 1.0) -> np.ndarray:
    """``x`` [T, H, D] rotated at integer ``positions`` [T] (exact turns: the
    angle of position p is p f, reduced in float64 from p f / 2 pi)."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    turns = np.asarray(positions, np.float64)[:, None] * (np.asarray(frequencies, np.float64) / (2 * np.pi))
    a = 2 * np.pi * (turns - np.round(turns))
    cs, sn = gain * np.cos(a)[:, None], gain * np.sin(a)[:, None]
    i1, i2 = (np.arange(0, dims, 2), np.arange(1, dims, 2)) if traditional else \
        (np.arange(dims // 2), np.arange(dims // 2, dims))
    y[..., i1] = x[..., i1] * cs - x[..., i2] * sn
    y[..., i2] = x[..., i1] * sn + x[..., i2] * cs
    return y


def pair_axes(pairs: int, sections=None, interleaved: bool = False) -> np.ndarray:
    """The axis that each pair turns by: in runs, or dealt in turn until an
    axis has its pairs (the first takes the rest)."""
    if sections is None:
        return np.zeros(pairs, int)
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections)
    left = list(sections)
    axis = np.zeros(pairs, int)
    for i in range(pairs):
        a = i % len(sections)
        if a and left[a]:
            axis[i] = a
            left[a] -= 1
    return axis


def norm_heads(x: np.ndarray, weight, eps: float) -> np.ndarray:
    """``x`` [T, H, D], each head over the root of its mean square, times ``weight``."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def rotate_axes(x: np.ndarray, positions, axis, frequencies, dims: int, traditional: bool, gain: float = 1.0) -> np.ndarray:
    """:func:`rotate` with ``positions`` [axes, T]: pair i turns by its own axis's."""
    y = np.array(x, np.float64)
    for a in range(len(positions)):
        r = rotate(x, positions[a], frequencies, dims, traditional, gain)
        for i in np.flatnonzero(np.asarray(axis) == a):
            for d in ((2 * i, 2 * i + 1) if traditional else (i, i + dims // 2)):
                y[..., d] = r[..., d]
    return y


def quantise_rows(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(int8 values, fp32 scale) of each row (last axis) of float32 ``x``."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(axis=-1)
    bad = ~np.isfinite(x).all(axis=-1)
    tiny = ~bad & (top < np.float32(2.0) ** -100)
    with np.errstate(all="ignore"):
        inv = np.where(bad | tiny, np.float32(0), np.float32(127) * (np.float32(1) / top))
        scale = np.where(bad, np.float32(np.nan), np.where(tiny, np.float32(0), top / np.float32(127)))
        q = np.rint(x * inv[..., None])
    return np.clip(np.nan_to_num(q, nan=0.0), -127, 127).astype(np.int8), scale.astype(np.float32)


def page_order(kind: str, head_dim: int, bits: int) -> np.ndarray:
    """[32, D] -> element of a 32-key block at which (key, d) is stored."""
    key, d = np.meshgrid(np.arange(32), np.arange(head_dim), indexing="ij")
    if kind == "k":
        n = 16 if bits == 8 else 8
        half, rest = d // (head_dim // 2), d % (head_dim // 2)
        return ((rest // n * 2 + half) * 32 + key) * n + rest % n
    jj, r = key // 16, key % 16
    half = r % 8 // 4
    e = np.where(r < 8, r % 4, 4 + r % 4)
    t, c = d // 32, d % 32
    if bits == 8:
        return ((t * 2 + half) * 32 + c) * 16 + jj * 8 + e
    return ((t * 2 + jj) * 64 + half * 32 + c) * 8 + e


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, start: int, scale: float | None = None,
           window: int | None = None, sinks: int = 0):
    """``q`` [n, Hq, D] at positions start.. over ``k``, ``v`` [Hkv, keys, D]:
    ``(o, spread, reach)`` float64: the rows, sum_j p_j |v_j| of each element,
    and per row max_j of sum_d |q_d k_jd| scale and of |score|. ``window``: the
    last so many positions up to a row's own, and the first ``sinks``."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, Hq, D = q.shape
    rep = Hq // k.shape[0]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, spread = np.zeros_like(q), np.zeros_like(q)
    reach = np.zeros((n, Hq))
    for i in range(n):
        seen = min(start + i + 1, k.shape[1])
        if seen <= 0:
            continue
        for h in range(Hq):
            kk, vv = k[h // rep, :seen], v[h // rep, :seen]
            if window is not None:
                j = np.arange(seen)
                j = j[(j > start + i - window) | (j < sinks)]
                if not len(j):
                    continue
                kk, vv = kk[j], vv[j]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h] = p @ vv
            spread[i, h] = p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return o, spread, reach
