"""Shared by the tests of the paged operators: random block tables, contents of
a cache as numbers, and the bounds that rounding allows.

Bounds. bf16 rounds by at most 2^-8 of a value (half a step), fp32 by 2^-24.
"""

import numpy as np
import torch

from oracle import paged as O

HALF = 2.0 ** -8   # bf16: half a step, relative


def rows(rng, *shape, scale=1.0):
    """bf16 rows on the GPU, a few columns larger than the others."""
    x = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[-1])) * scale
    return torch.from_numpy(x.astype(np.float32)).cuda().to(torch.bfloat16)


def num(t):
    return t.detach().double().cpu().numpy()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables(rng, lengths, page, extra=2):
    """(block table [B, width] with -1 where there is no page, pages in all),
    pages in random order."""
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + extra
    order = rng.permutation(pages)
    t = np.full((len(lengths), max(1, max(used))), -1, np.int32)
    at = 0
    for b, n in enumerate(used):
        t[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(t).cuda(), pages


def stored(cache, table, b, count):
    """float64 (K, V) [Hkv, count, D] that request b's first `count` positions
    hold, from the raw pages and the order that the oracle gives."""
    out = []
    for kind, pages, scales in (("k", cache.k_pages, cache.k_scales), ("v", cache.v_pages, cache.v_scales)):
        at = O.page_order(kind, cache.head_dim, cache.bits).reshape(-1)
        nb = -(-count // cache.page_size)
        ids = table[b, :nb].long()
        raw = num(pages[ids])                                   # [nb, H, page / 32, 32 D]
        x = raw[..., at].reshape(raw.shape[:3] + (32, cache.head_dim))
        x = x.transpose(1, 0, 2, 3, 4).reshape(cache.n_kv_heads, -1, cache.head_dim)
        if scales is not None:
            s = num(scales[ids]).transpose(1, 0, 2).reshape(cache.n_kv_heads, -1)
            with np.errstate(invalid="ignore"):
                x = x * s[..., None]
        out.append(x[:, :count])
    return out


def attention_bound(o, spread, reach, head_dim):
    """How far bf16 attention may be from float64 on the same numbers.

    * the output's rounding: 2^-8 |o|;
    * each weight is rounded once to bf16 (their sum is not): 2^-8 sum p |v|;
    * a score is an fp32 sum of D products (D 2^-24 of sum |q k| scale), takes
      up to four fp32 roundings more (scale, key scale, maximum, exponent's
      argument: 2^-22 of it), and moves its weight by that much relatively; the
      maximum's row likewise, so twice;
    * the exponential itself, sums of weights and of products in fp32 over
      chains of a few thousand: 2^-14, generously.
    """
    eta = 2 * reach * (head_dim * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -14
    return HALF * np.abs(o) * 1.01 + (HALF * 1.01 + eta[..., None]) * spread


def check_rows(got, want, bound, what):
    err = np.abs(got - want)
    bad = ~(err <= bound + 1e-30)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} out of bounds; first at {i}: got {got[i]}, "
                             f"want {want[i]} +- {bound[i]}")
