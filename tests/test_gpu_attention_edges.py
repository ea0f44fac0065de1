"""GPU: attention over the paged cache at the ends of what it admits, against the definition in 64 bits."""
import math

import pytest
import torch

from tests._attention import attend as reference, check_out
from tests.test_gpu_attention import BF16, F16, check, make, run
from valora_amd.attention import AttentionPlan

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


def probabilities(c, b, page, window=0):
    """``(weights [new, heads, cached] of request b's rows, what each sees [new, cached])`` in 64 bits; nan where the row's q is."""
    n, length, at = c["news"][b], c["lens"][b], c["starts"][b]
    j = torch.arange(length)
    pages = c["table"][b].long()[j // page]
    ok = (pages >= 0) & (pages < c["kb"].shape[0] // page)
    rows = torch.where(ok, pages, torch.zeros_like(pages)) * page + j % page
    p = torch.arange(length - n, length)[:, None]
    sees = (j[None] <= p) & ok[None]
    if window:
        sees = sees & (j[None] > p - window)
    hq, hkv, d = c["q"].shape[1], c["kb"].shape[1], c["q"].shape[2]
    out = torch.zeros(n, hq, length, dtype=torch.float64)
    for h in range(hq):
        s = c["q"][at:at + n, h].double() @ c["kb"][rows, h // (hq // hkv)].double().T * d ** -0.5
        s = torch.where(sees, s, torch.full_like(s, -math.inf))
        # (a row that sees nothing, or whose scores are all -infinity, gives no weight)
        out[:, h] = torch.where((s == -math.inf).all(-1, keepdim=True), torch.zeros_like(s), torch.softmax(s, -1))
    return out, sees


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("n,length,window", [(3, 40, 0), (4, 300, 7), (2, 700, 0), (1, 90, 0), (20, 60, 0), (60, 700, 9)])
def test_weights_of_a_row_that_is_no_number(dev, n, length, window, value):
    """It makes the weights of what it sees no numbers, and leaves those of later tokens, of tokens behind its window and of tokens whose
    page is not there as the other rows make them; few rows and tall tiles alike."""
    page, hq, hkv = 4, 4, 2
    c = make(dev, BF16, hq, hkv, 64, page, [(n, length), (1, 30)], seed=32)
    c["q"][0, 1, 5] = value                              # the first row of the first request
    c["table"][0, 2], c["table"][0, (length - n) // page - 1] = -1, 2**30
    w = torch.zeros(2, c["table"].shape[1] * page, device=dev)
    run(dev, c, page, window, weights=w)
    p, sees = probabilities(c, 0, page, window)
    bad = ~torch.isfinite(p).all(-1)                     # [new, heads]
    # (infinity times the three keys that the row of the window of 7 sees: -infinity each)
    assert int(bad.sum()) == (0 if value == math.inf and window == 7 else 1)
    poisoned = sees[0] & bad.any()
    want = torch.where(bad[:, :, None], torch.zeros_like(p), p).sum((0, 1))
    got = w[0, :length].cpu().double()
    assert bool(torch.isnan(got[poisoned]).all())
    assert int((~poisoned).sum()) >= 8 and not got[8:12].any()
    # scores in 32 bits, of 64 products whose sizes add up to less than 16: off by 2 * 64 * 2^-24 * 16, as is a row's logarithm
    assert torch.allclose(got[~poisoned], want[~poisoned], rtol=2.0 ** -11, atol=2.0 ** -30)
    p1, _ = probabilities(c, 1, page, window)
    assert torch.allclose(w[1, :30].cpu().double(), p1.sum((0, 1)), rtol=2.0 ** -11, atol=2.0 ** -30)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("gap", [7.0, 12.0, 16.0, 18.0, 20.0])
@pytest.mark.parametrize("n,n_req", [(1, 64), (20, 32)])
def test_one_token_far_above_a_long_tail_in_fp16(dev, n, n_req, gap, first):
    """One token's score lies `gap` above those of tens of thousands, whose weights together count all the same, in requests enough that a
    wave has thousands of them beside it.  Weights keep their eleven bits down to 2^-21 of the largest and are off by at most 2^-32 of
    it below: 2^7 of the 2^15 that fp16 goes to are used when the reference is set."""
    length, heads, d = 60000, 16, 32
    g = torch.Generator().manual_seed(33)
    q = torch.zeros(n * n_req, heads, d, dtype=F16)
    q[:, :, 0] = 8.0
    kb = torch.zeros(length, heads, d, dtype=F16)
    vb = (0.5 + torch.rand(length, heads, d, generator=g)).to(F16)
    top = 0 if first else length - n
    kb[top, :, 0] = gap                                  # 8 * gap / 8
    vb[top] = 0
    table = torch.arange(length, dtype=torch.int32).expand(n_req, length).contiguous()       # (all look at the same cache)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    plan = AttentionPlan(i32(list(range(0, n * n_req, n))), i32([n] * n_req), i32([length] * n_req), n_tokens=n * n_req, max_seq_len=n,
                         max_kv_len=length, q_heads=heads, kv_heads=heads, head_dim=d)
    got = plan.attend(torch.full_like(q, 7.0, device=dev), q.to(dev), kb.to(dev), vb.to(dev), table.to(dev), scale=0.125)
    want, _, bound, _ = reference(q[:n], kb, vb, table, [0], [n], [length], 1, 0, 0.125)
    # (the general bound allows 2^-25 of the largest weight a token: it knows of no reference below the maximum)
    bound = bound - 2 * length * (2.0 ** -25 - 2.0 ** -32) * float(vb.abs().max())
    assert bool((bound > 0).all())
    for b in range(n_req):
        check_out(got[b * n:(b + 1) * n], want, bound, f"request {b}")


@pytest.mark.parametrize("n,length", [(1, 3000), (1, 100), (40, 700), (130, 4000)])
def test_bf16_values_as_large_as_the_type_holds(dev, n, length):
    """Their mean over many tokens is no larger than they are."""
    big = torch.finfo(BF16).max
    c = make(dev, BF16, 2, 1, 64, 1, [(n, length)], seed=35)
    c["q"][:, 0] = 0                                     # a head that looks at all alike, and one that does not
    c["vb"][:, :, :32], c["vb"][:, :, 32:] = big, -big
    got = run(dev, c, 1).cpu().double()
    want = torch.full_like(got, big)
    want[:, :, 32:] = -big
    # a rounding to bf16, sums in 32 bits
    assert bool(((got - want).abs() <= (2.0 ** -8 + (length + 64) * 2.0 ** -24) * big).all()), float((got - want).abs().max() / big)


@pytest.mark.parametrize("dtype,size", [(F16, 8000.0), (F16, 65504.0), (BF16, 1e6), (BF16, 1e15)])
@pytest.mark.parametrize("n,length", [(1, 90), (1, 3000), (40, 700), (130, 4000)])
def test_scores_far_beyond_what_32_bits_resolve(dev, dtype, size, n, length):
    """Equal ones give the mean; of unequal ones the highest takes all; and no weight is more than a row has."""
    d = 128
    c = make(dev, dtype, 2, 1, d, 1, [(n, length)], seed=36)
    c["q"][:], c["kb"][:] = size, size
    u = torch.finfo(dtype).eps / 2
    rows = c["table"][0].long()[:length]
    w = torch.zeros(1, c["table"].shape[1], device=dev)
    got = run(dev, c, 1, weights=w).cpu().double()
    V = c["vb"][rows, 0].double()
    mean = V.cumsum(0) / torch.arange(1, length + 1)[:, None]
    # all scores are the same number, so all weights are: what is left is the sums' rounding and the result's
    err = (got - mean[length - n:, None]).abs()
    assert bool((err <= u * mean[length - n:, None].abs() + 2 * (length + 64) * 2.0 ** -24 * float(V.abs().max())).all()), float(err.max())
    assert bool(torch.isfinite(w).all()) and float(w.max()) <= 2 * n * (1 + 2.0 ** -10)
    # each token's key a step of the type above or below the last one's: the highest is the row's last, or its first
    step = torch.arange(length) % 64 * (4 * u)
    for sign in (1.0, -1.0):
        c["kb"][rows, 0] = (size / 2 * (1 + sign * step))[:, None].to(dtype).expand(length, d)
        got = run(dev, c, 1, weights=w).cpu().double()
        k = c["kb"][rows, 0, 0].double()
        for i in range(n):
            best = k[:length - n + i + 1] == k[:length - n + i + 1].max()
            want = V[:length - n + i + 1][best].mean(0)
            assert bool(((got[i] - want).abs() <= u * want.abs() + 2 * (length + 64) * 2.0 ** -24 * float(V.abs().max())).all()), (sign, i)
        assert bool(torch.isfinite(w).all()) and float(w.max()) <= 6 * n * (1 + 2.0 ** -10)
