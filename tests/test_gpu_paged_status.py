"""The paged cache's status word, with calls in flight on other streams."""

import numpy as np
import pytest
import torch

from mtplx_amd import _lib
from mtplx_amd.paged_kv_cache import PagedKVCache
from tests.paged_util import i32, rows

pytestmark = pytest.mark.gpu


def test_check_status_sees_other_streams(gpu):
    """A write without a page, behind work on a stream that the current one does
    not wait for: the check sees it, and clears it once."""
    rng = np.random.default_rng(41)
    c = PagedKVCache(2, 1, 64, page_size=32)
    x, table, start = rows(rng, 4, 1, 64), i32([[-1]]), i32([0])
    a = torch.randn((4096, 4096), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.check_status()
    for _ in range(3):
        with torch.cuda.stream(side):
            for _ in range(20):   # some milliseconds
                a @ a
            c.write(x, x, table, start)
        with pytest.raises(_lib.MtpError):
            c.check_status()
        torch.cuda.synchronize()
        assert int(c.status().item()) == 0
        c.check_status()
