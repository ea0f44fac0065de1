"""GPU: attention over the paged cache at the ends of what it admits, against the definition in 64 bits."""
import math

import pytest
import torch

from tests._attention import attend as reference, check_out
from tests.test_gpu_attention import BF16, F16, check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 20, 2**30 + 1, 1000])
@pytest.mark.parametrize("reqs", [[(5, 2), (3, 3), (1, 9)], [(40, 10), (200, 100), (300, 900), (2, 1)]])
def test_windows_beyond_any_cache(dev, window, reqs):
    """They bound nothing, also where the first rows lie before the cache's first token."""
    for dtype, hq in ((F16, 4), (BF16, 2)):
        c = make(dev, dtype, hq, 2, 64, 1, reqs, seed=31)
        w = torch.zeros(len(reqs), c["table"].shape[1], device=dev)
        got, want, w_bound = check(dev, c, 1, window, weights=w)
        check_out(w, want, w_bound + 2.0 ** -60)
        assert torch.equal(run(dev, c, 1, 0), got)
