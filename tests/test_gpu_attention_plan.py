"""GPU: batches for which the plan kernel goes round more than once: more requests, and more tall tiles, than it has threads (512)."""
import random

import pytest
import torch

from tests._attention import check_out
from tests.test_gpu_attention import BF16, F16, check, make

pytestmark = pytest.mark.gpu


def batch(n_req, news, longest, seed):
    """Requests of the new tokens `news` in turn, empty ones among them, few of them long."""
    rng = random.Random(seed)
    out = []
    for i in range(n_req):
        n = news[i % len(news)]
        length = n + (rng.randint(longest // 2, longest) if rng.random() < 0.03 else rng.randint(0, 60))
        out.append((0 if rng.random() < 0.05 else n, min(length, longest)))
    return out


@pytest.mark.parametrize("window", [0, 23])
@pytest.mark.parametrize("news,longest", [([1], 120), ([1, 2], 900), ([5], 400), ([5, 9], 900), ([1, 5, 1, 40], 700), ([1, 40, 3], 300)])
def test_more_requests_and_tiles_than_threads(dev, news, longest, window):
    """Decoding requests whole and cut, tall tiles (more than 16 rows of 4 heads) each a share and in a line, both mixed."""
    reqs = batch(1300, news, longest, seed=len(news) + longest)
    tiles = sum(-(-n * 4 // 128) for n, _ in reqs if n * 4 > 16)
    assert max(l for _, l in reqs) > longest // 2 and (tiles > 512 or max(news) * 4 <= 16)
    c = make(dev, BF16 if window else F16, 4, 1, 32, 1, reqs, seed=37, gap=1)
    w = torch.zeros(len(reqs), c["table"].shape[1], device=dev)
    _, want, w_bound = check(dev, c, 1, window, weights=w)
    check_out(w, want, w_bound + 2.0 ** -60)
