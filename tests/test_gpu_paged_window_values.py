"""Values that are no numbers behind a window at every head dim: the rows that do not
see them keep their bits, those that do show them (chunks flag such blocks as they
are staged, each head dim in a ring of its own)."""

import numpy as np
import pytest
import torch

from mtplx_amd.paged_attention import paged_sdpa
from mtplx_amd.paged_kv_cache import PagedKVCache
from tests.paged_util import i32, rows
from tests.test_gpu_paged_attention import _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,keys,window,sinks", [(3, 700, 200, 5), (330, 1500, 200, 5), (330, 1500, 600, 0)])
def test_values_behind_a_window(gpu, D, bits, n, keys, window, sinks):
    rng = np.random.default_rng(D + bits + n)
    c, table = _filled(rng, [keys], D, 1, 32, bits)
    q = rows(rng, n, 4, D)
    start = keys - n
    kw = dict(window=window, sinks=sinks)
    want = paged_sdpa(q, c, table, i32([start]), **kw)
    assert torch.isfinite(want).all()
    pos = start + np.arange(n)
    for at in (2, 31, start - window, start - window + 1, start - window + 130, start - 1, start + n // 2, keys - 1):
        d = PagedKVCache(c.num_pages, 1, D, page_size=32, bits=bits)
        for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
            if getattr(c, name) is not None:
                getattr(d, name).copy_(getattr(c, name))
        bad = rows(rng, 1, 1, D)
        bad[0, 0, D // 2 + 1] = float("nan")
        d.write(torch.zeros_like(bad), bad, table, i32([at]))
        got = paged_sdpa(q, d, table, i32([start]), **kw)
        seen = torch.from_numpy((at <= pos) & ((at > pos - window) | (at < sinks))).cuda()
        assert torch.equal(got[~seen], want[~seen]), at
        assert torch.isnan(got[seen][..., D // 2 + 1]).all(), at
