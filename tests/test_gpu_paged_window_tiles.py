"""Windowed prompts whose tiles fall to workgroups whole, one or several each, and ones
that are cut, with float64 attention over what the pages hold at rows of every tile's
ends."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from tests.paged_util import i32, rows
from tests.test_gpu_paged_attention import _filled
from tests.test_gpu_paged_window import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,Hq,H,D,bits,window,sinks", [
    (4000, 16, 4, 64, 16, 256, 0), (4000, 16, 4, 64, 8, 250, 7),     # one whole tile each
    (8192, 16, 4, 64, 16, 512, 0),                                  # two
    (4000, 24, 4, 256, 16, 256, 0), (8192, 40, 8, 128, 8, 512, 4),   # three and five
    (5000, 40, 8, 128, 16, 1024, 0), (4000, 16, 4, 64, 16, 1024, 3),   # cut
])
def test_whole_and_cut_tiles(gpu, n, Hq, H, D, bits, window, sinks):
    rng = np.random.default_rng(n + D + window)
    c, table = _filled(rng, [n], D, H, 64, bits)
    q = rows(rng, n, Hq, D)
    got = paged_sdpa(q, c, table, i32([0]), window=window, sinks=sinks)
    assert torch.isfinite(got).all()
    tile = (128 if D == 256 else 256) * H // Hq
    check(c, table, q, [n], [n], got, window, sinks, what=str(n),
          rows_of=lambda m: sorted({0, 1, window - 1, window, m - 2, m - 1, *range(0, m, 7 * tile), *range(tile - 1, m, 9 * tile)}))
    assert torch.equal(got, paged_sdpa(q, c, table, i32([0]), window=window, sinks=sinks))


def test_no_rows_at_all(gpu):
    """Requests of no rows: nothing is written."""
    c, table = _filled(np.random.default_rng(1), [64, 64], 64, 1, 32, 16)
    q = rows(np.random.default_rng(2), 300, 2, 64)
    out = torch.full_like(q, 5.0)
    for max_rows in (None, 1):
        paged_sdpa(q, c, table, i32([63, 63]), i32([0, 0, 0]), max_rows=max_rows, window=9, sinks=2, out=out)
        assert (out == 5).all()
