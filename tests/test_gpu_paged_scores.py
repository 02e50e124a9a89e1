"""paged_sdpa where scores are infinite or weights nothing: what softmax over
the keys that a row sees gives, at every place of a row's keys (blocks with and
without a mask, pieces of one tile in several workgroups)."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from oracle import paged as O
from tests.paged_util import attention_bound, check_rows, i32, num, rows, stored, tables

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 40), (4, 900), (40, 40), (90, 300), (70, 5000)]   # new tokens, keys


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,keys", SHAPES)
def test_scores_of_minus_infinity(gpu, n, keys, D):
    """Keys of score -infinity have weight 0; a row that sees no other is NaN, as
    softmax is; a row that sees no key at all is zeros."""
    rng = np.random.default_rng(n + keys + D)
    H, Hq = 2, 4
    for what in ("all", "first", "last", "most"):
        table, pages = tables(rng, [keys], 64)
        c = PagedKVCache(pages, H, D, page_size=64)
        k, v, q = rows(rng, keys, H, D), rows(rng, keys, H, D), rows(rng, n, Hq, D)
        gone = {"all": slice(0, keys), "first": slice(0, keys - (n + 1) // 2), "last": slice(keys - n // 2 - 1, keys),
                "most": slice(0, max(keys - 1, 1))}[what]
        q[..., 5] = 1.0
        k[gone, :, 5] = float("-inf")
        c.write(k, v, table, i32([0]))
        o, spread = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
        dead = np.zeros(n, bool)
        kv = stored(c, table, 0, keys)
        for i in range(n):   # over the keys whose score is finite
            seen = np.arange(keys - n + i + 1)
            seen = seen[(seen < gone.start) | (seen >= gone.stop)]
            dead[i] = not len(seen)
            if not dead[i]:
                r = O.attend(num(q[i:i + 1]), *(x[:, seen] for x in kv), len(seen) - 1)
                o[i], spread[i] = r[0][0], attention_bound(*r, D)[0]
        for kw in (dict(), dict(row_off=i32([0, n]))):
            got = num(paged_sdpa(q, c, table, i32([keys - n]), **kw))
            check_rows(got[~dead], o[~dead], spread[~dead], f"{what} {kw}")
            assert np.isnan(got[dead]).all(), f"{what} {kw}"
        assert (num(paged_sdpa(q, c, table, i32([-n]))) == 0).all()
        assert (num(paged_sdpa(q, c, torch.full_like(table, -1), i32([keys - n]))) == 0).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,keys,D", [(4, 140, 128), (40, 140, 128), (70, 300, 64), (40, 140, 256), (4, 140, 256)])
def test_a_value_that_is_no_number_at_a_weight_of_nothing(gpu, n, keys, D, bits):
    """NaN in a value whose key's weight underflows: the rows that see it show it
    (0 times NaN), wherever it lies; those before it keep their bits."""
    rng = np.random.default_rng(n + D + bits)
    table, pages = tables(rng, [keys], 64)
    k, v, q = rows(rng, keys, 1, D, scale=0.1), rows(rng, keys, 1, D), rows(rng, n, 2, D, scale=0.1) + 2
    for at in (5, 70, keys - n + 1, keys - 2, keys - 1):
        kk, vv, plain = k.clone(), v.clone(), []
        kk[at] = -400.0   # scores of -6400 and less
        for value in (0.0, float("nan")):
            vv[at, 0, 3] = value
            c = PagedKVCache(pages, 1, D, page_size=64, bits=bits)
            c.write(kk, vv, table, i32([0]))
            for kw in (dict(), dict(row_off=i32([0, n]))):
                plain.append(num(paged_sdpa(q, c, table, i32([keys - n]), **kw)))
        first = max(at - (keys - n), 0)
        for good, got in zip(plain[:2], plain[2:]):
            assert np.isfinite(good).all() and np.array_equal(got[:first], good[:first])
            assert np.isnan(got[first:, :, 3]).all(), at
            if bits == 8:
                assert np.isnan(got[first:]).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [4, 90])
def test_large_values(gpu, n, bits):
    """Sums are not normalised until the end: values of 2^100 over 1000 keys stay
    within 2^120, and a power of two changes no bit of what it scales."""
    rng = np.random.default_rng(n + bits)
    keys, H, D = 1000, 2, 128
    table, pages = tables(rng, [keys], 64)
    k, v, q = rows(rng, keys, H, D), rows(rng, keys, H, D), rows(rng, n, 4, D)
    got = []
    for scale in (1.0, 2.0 ** 100):
        c = PagedKVCache(pages, H, D, page_size=64, bits=bits)
        c.write(k, v * scale, table, i32([0]))
        got.append(num(paged_sdpa(q, c, table, i32([keys - n]))) / scale)
    assert np.isfinite(got[0]).all() and np.array_equal(*got)
