"""The marked values of the long attention tests (CPU): deleting or doubling any
32-key block of the longest row moves some element past the bound."""

import numpy as np
import pytest

from oracle import paged as O
from tests.paged_util import HALF


@pytest.mark.parametrize("keys,D", [(40000, 64), (40000, 128), (20064, 256), (30000, 128)])
def test_every_block_shows(keys, D):
    rng = np.random.default_rng(keys + D)
    wide = lambda n, scale: rng.standard_normal((n, D)) * np.exp(0.5 * rng.standard_normal(D)) * scale  # noqa: E731
    k, q = wide(keys, 1.0), wide(1, 0.2)
    s = k @ q[0] / np.sqrt(D)
    p = np.exp(s - s.max())
    block = np.arange(keys) // 32
    blocks = np.bincount(block, weights=p)          # weight of each block
    column = np.bincount(np.arange(len(blocks)) % D, weights=blocks, minlength=D)
    reach = (np.abs(k) @ np.abs(q[0])).max() / np.sqrt(D)
    eta = 2.02 * HALF + 2 * reach * (D * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -14
    for i, w in enumerate(blocks):
        have, total = column[i % D] / p.sum(), p.sum()
        for sign in (-1, 1):
            got = (column[i % D] + sign * w) / (total + sign * w)
            assert abs(got - have) > 1.5 * eta * have, i
    o, spread, _ = O.attend(q[None], k[None], np.eye(D)[block % D][None], keys - 1)   # the oracle's own numbers
    assert np.allclose(o[0, 0], column / p.sum()) and np.array_equal(o, spread)
