"""GPU: attention over the 8-bit cache.  Its values are exact in the tensors' type, so the definition and the bounds are those of the 16-bit
cache that holds them (tests/_attention.py)."""
import math

import pytest
import torch

from tests._attention import attend as reference, check_out
from tests._cache8 import cache_of, pages_of
from tests.test_gpu_attention import LONG, MIXED, make
from valora_amd.attention import AttentionPlan

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def coded(dev, page, *a, small=1.0, **kw):
    """A case of the 16-bit tests, its cache as codes; the definition takes the values they stand for."""
    dtype = a[0]
    c = make(dev, *a[:4], page, *a[4:], **kw)
    c["key_codes"], c["value_codes"], c["powers"], c["kb"], c["vb"] = cache_of(c["kb"].double() * small, c["vb"].double() * small, page, dtype)
    return c


def run(dev, c, page, window=0, scale=None, weights=None, out=None, max_seq=None, max_kv=None, plan=None):
    hq, d, hkv = c["q"].shape[1], c["q"].shape[2], c["kb"].shape[1]
    if plan is None:
        plan = AttentionPlan(*c["lengths"], n_tokens=c["T"], max_seq_len=max(c["news"] + [0]) if max_seq is None else max_seq,
                             max_kv_len=max(c["lens"] + [0]) if max_kv is None else max_kv, q_heads=hq, kv_heads=hkv, head_dim=d,
                             page_size=page, window=window)
    if out is None:
        out = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device=dev)
    plan.attend8(out, c["q"].to(dev), c["key_codes"].to(dev), c["value_codes"].to(dev), c["powers"].to(dev), c["table"].to(dev), scale=scale,
                 weights=weights)
    torch.cuda.synchronize()
    return out


def check(dev, c, page, window=0, scale=None, **kw):
    want, weights, bound, w_bound = reference(c["q"], c["kb"], c["vb"], c["table"], c["starts"], c["news"], c["lens"], page, window,
                                              c["q"].shape[2] ** -0.5 if scale is None else scale, max_kv=kw.get("max_kv"))
    got = run(dev, c, page, window, scale, **kw)
    check_out(got, want, bound)
    left = torch.isnan(bound)
    assert bool((got.cpu()[left] == 7.0).all()), "rows of no request"
    return got, weights, w_bound


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (28, 4, 64), (6, 2, 96), (4, 4, 32), (2, 1, 256), (16, 1, 256)])
@pytest.mark.parametrize("page", [2, 16])
def test_heads_and_lengths(dev, dtype, hq, hkv, d, page):
    check(dev, coded(dev, page, dtype, hq, hkv, d, LONG, seed=1, gap=1), page)
    check(dev, coded(dev, page, dtype, hq, hkv, d, MIXED, seed=2, gap=2), page)


@pytest.mark.parametrize("n", [1, 2, 4, 5, 16, 17, 32, 33, 64, 127, 128, 129, 260])
def test_new_tokens_around_the_tiles(dev, n):
    check(dev, coded(dev, 2, BF16, 4, 1, 64, [(n, n), (n, n + 63), (n, n + 64), (n, n + 65), (n, n + 511)], seed=n), 2)
    check(dev, coded(dev, 1, F16, 4, 1, 32, [(n, n), (n, n + 63), (n, n + 64), (n, n + 65), (n, n + 511)], seed=n), 1)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 128, 256])
def test_pages_that_end_inside_a_tile(dev, page):
    """What no request's token owns is no number."""
    check(dev, coded(dev, page, F16, 4, 2, 64, [(1, 77), (3, 130), (40, 300), (1, 256), (1, 257)], seed=page, fill=math.nan), page)
    check(dev, coded(dev, page, BF16, 2, 2, 96, [(1, 77), (3, 130), (40, 300), (1, 256), (1, 257)], seed=page, fill=math.nan), page)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
def test_window(dev, window):
    reqs = [(1, 1), (1, 64), (1, 777), (5, 300), (90, 90), (130, 900), (16, 16)]
    check(dev, coded(dev, 2, BF16, 8, 4, 64, reqs, seed=window), 2, window)
    check(dev, coded(dev, 16, F16, 4, 4, 128, reqs, seed=window + 1), 16, window)


@pytest.mark.parametrize("pieces", [(1, 20000, 1, 1), (40, 9000, 1, 1), (1, 5000, 4, 1), (300, 8200, 8, 1)])
def test_long_caches_in_many_pieces(dev, pieces):
    n, length, hq, hkv = pieces
    check(dev, coded(dev, 2, BF16, hq, hkv, 64, [(n, length)], seed=3, sharp=2.0), 2)


def test_rows_that_see_nothing_become_zeros(dev):
    c = coded(dev, 2, F16, 4, 2, 64, [(5, 2), (3, 0), (40, 7), (1, 0), (200, 100)], seed=4)
    got, _, _ = check(dev, c, 2)
    for b, (n, l) in enumerate(zip(c["news"], c["lens"])):
        assert not got[c["starts"][b]:c["starts"][b] + n - l].any()
    check(dev, c, 2, window=3)
    check(dev, coded(dev, 16, BF16, 1, 1, 128, [(0, 0), (2, 0)], seed=5), 16)


@pytest.mark.parametrize("d", [64, 256])
def test_pages_outside_the_pool_are_seen_by_no_one(dev, d):
    for n_new in (1, 50):
        c = coded(dev, 16, BF16, 4, 2, d, [(n_new, 200), (n_new, 90), (n_new, 64)], seed=6)
        c["key_codes"].view(torch.uint8)[0], c["value_codes"].view(torch.uint8)[0] = 127, 255   # what stands in for them must not show
        c["powers"].view(torch.uint8)[0] = 255
        c["kb"][0:16], c["vb"][0:16] = math.nan, math.nan
        c["table"][c["table"] == 0] = 1_000_000
        c["table"][0, 3], c["table"][0, 5] = -1, -2**31
        c["table"][1, :] = 2**31 - 1
        got, _, _ = check(dev, c, 16)
        at = c["starts"][1]
        assert not got[at:at + n_new].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,length", [(9, 40), (60, 60), (130, 400)])
@pytest.mark.parametrize("value", [math.nan, math.inf, "max"])
def test_what_a_row_does_not_see_does_not_show(dev, dtype, n, length, value):
    """Later tokens, tokens behind the window and the rest of the last page hold no numbers, or the largest; rows that see one follow the
    arithmetic.  (An infinity becomes the largest value when it is coded.)"""
    value = torch.finfo(dtype).max if value == "max" else value
    for window in (0, 11):
        c = make(dev, dtype, 4, 2, 64, 16, [(n, length)], seed=7, fill=value)
        j = length - 3
        row = int(c["table"][0, j // 16]) * 16 + j % 16
        c["vb"][row, 0, 5] = value
        c["vb"][row, 1, :] = value
        c["key_codes"], c["value_codes"], c["powers"], c["kb"], c["vb"] = cache_of(c["kb"], c["vb"], 16, dtype)
        check(dev, c, 16, window)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 16, 16, 128), (BF16, 32, 16, 128), (BF16, 16, 16, 64), (F16, 16, 8, 256)])
@pytest.mark.parametrize("value", [math.nan, math.inf, "max"])
def test_many_requests_that_decode(dev, dtype, hq, hkv, d, value):
    """More requests times key heads than a list is cut for, each several tiles of a wave long; some see values that are no numbers, or the
    largest, early and late."""
    value = torch.finfo(dtype).max if value == "max" else value
    reqs = [(1, 1 + 37 * i % 701) for i in range(130 if hkv == 8 else 70)]
    c = make(dev, dtype, hq, hkv, d, 2, reqs, seed=13)
    for b in range(0, len(reqs), 5):
        for j in (reqs[b][1] // 7, reqs[b][1] - 1):
            row = int(c["table"][b, j // 2]) * 2 + j % 2
            c["vb"][row, b % hkv, j % d] = value
            c["vb"][row, (b + 1) % hkv, :] = value
    c["key_codes"], c["value_codes"], c["powers"], c["kb"], c["vb"] = cache_of(c["kb"], c["vb"], 2, dtype)
    check(dev, c, 2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("byte", [0, 255])
def test_powers_that_were_never_written(dev, dtype, byte):
    """Beside tokens that no row sees yet: any byte may stand there."""
    c = coded(dev, 16, dtype, 4, 2, 128, [(1, 40), (33, 70)], seed=8)
    owned = torch.zeros(c["kb"].shape[0], dtype=torch.bool)
    for b, l in enumerate(c["lens"]):
        j = torch.arange(l)
        owned[c["table"][b].long()[j // 16] * 16 + j % 16] = True
    free = pages_of((~owned)[:, None].expand(-1, 2), 16)
    c["powers"].view(torch.uint8)[free] = byte
    check(dev, c, 16)


@pytest.mark.parametrize("dtype,small", [(F16, 2.0 ** -14), (F16, 2.0 ** 5), (BF16, 2.0 ** -40), (BF16, 2.0 ** 40)])
def test_small_and_large_values(dev, dtype, small):
    """Powers far from 1, for k and v alike; the scale keeps the scores within reach."""
    c = coded(dev, 2, dtype, 4, 2, 64, [(1, 90), (20, 150)], seed=9, small=small)
    check(dev, c, 2, scale=0.125 / small)


def test_strides(dev):
    """Keys' and values' pages side by side in one tensor, rows of q and out within wider ones, powers in a wider tensor."""
    page, hkv, d = 4, 2, 64
    c = coded(dev, page, BF16, 4, hkv, d, [(1, 50), (30, 61), (2, 9)], seed=10, gap=1)
    n = c["key_codes"].shape[0]
    both = torch.stack([c["key_codes"].view(torch.uint8), c["value_codes"].view(torch.uint8)], 1).to(dev).view(torch.float8_e4m3fn)
    wide = torch.zeros(n, hkv * page * 2 + 6, dtype=torch.uint8, device=dev)
    wide[:, :hkv * page * 2] = c["powers"].view(torch.uint8).flatten(1).to(dev)
    powers = wide[:, :hkv * page * 2].unflatten(1, (hkv, page, 2)).view(torch.float8_e8m0fnu)
    q = torch.zeros(c["T"], 4 * d + 8, dtype=BF16, device=dev)
    q[:, :4 * d] = c["q"].to(dev).flatten(1)
    out = torch.full((c["T"], 5, d), 7.0, dtype=BF16, device=dev)
    plan = AttentionPlan(*c["lengths"], n_tokens=c["T"], max_seq_len=30, max_kv_len=61, q_heads=4, kv_heads=hkv, head_dim=d, page_size=page)
    plan.attend8(out[:, :4], q[:, :4 * d], both[:, 0], both[:, 1], powers, c["table"].to(dev))
    want, _, bound, _ = reference(c["q"], c["kb"], c["vb"], c["table"], c["starts"], c["news"], c["lens"], page, 0, d ** -0.5)
    check_out(out[:, :4], want, bound)
    assert bool((out[:, 4] == 7.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,page", [(128, 2), (64, 16), (256, 1), (96, 4), (32, 2)])
@pytest.mark.parametrize("reqs", [[(1, 400), (2, 90), (1, 1)], [(40, 300), (1, 500), (3, 3)]])
def test_weights(dev, dtype, d, page, reqs):
    c = coded(dev, page, dtype, 4, 2, d, reqs, seed=11)
    w = torch.rand(len(reqs), c["table"].shape[1] * page, generator=torch.Generator().manual_seed(1)).to(dev)
    before = w.cpu().double()
    _, want, bound = check(dev, c, page, weights=w)
    err = (w.cpu().double() - before - want).abs()
    assert bool((err <= bound + 2.0 ** -22).all()), float((err - bound).max())


def test_no_result_depends_on_the_split(dev):
    """The same requests alone and in a batch, and the same call twice: the second gives the same bits."""
    c = coded(dev, 2, F16, 8, 2, 128, [(1, 3000), (1, 40), (64, 900)], seed=12)
    a, b = run(dev, c, 2), run(dev, c, 2)
    assert torch.equal(a, b)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (10, 5), (24, 3), (16, 16)])
@pytest.mark.parametrize("window", [0, 70])
def test_weights_of_prompts_by_heads(dev, hq, hkv, window):
    """Heads fewer and more than the waves that share them out, rows that do not divide."""
    reqs = [(37, 300), (130, 130), (1, 200), (3, 70), (66, 65)]
    c = coded(dev, 2, BF16, hq, hkv, 64, reqs, seed=13)
    w = torch.zeros(len(reqs), c["table"].shape[1] * 2, device=dev)
    _, want, bound = check(dev, c, 2, window, weights=w)
    err = (w.cpu().double() - want).abs()
    assert bool((err <= bound + 2.0 ** -22).all()), float((err - bound).max())


def test_weights_where_the_scores_have_no_room(dev):
    """More scores than the workspace's bound: the keys are read a second time."""
    n, length = 200, 20000
    g = torch.Generator(device="cpu").manual_seed(14)
    hq, hkv, d, page = 32, 4, 32, 64
    pages = 400
    kb, vb = torch.randn(pages * page, hkv, d, generator=g), torch.randn(pages * page, hkv, d, generator=g)
    kc, vc, powers, k, v = cache_of(kb, vb, page, BF16)
    table = torch.randint(0, pages, (n, -(-length // page)), generator=g).to(torch.int32)
    q = torch.randn(n, hq, d, generator=g).to(BF16)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    plan = AttentionPlan(i32(range(n)), i32([1] * n), i32([length] * n), n_tokens=n, max_seq_len=1, max_kv_len=length, q_heads=hq, kv_heads=hkv,
                         head_dim=d, page_size=page)
    w = torch.zeros(n, length, device=dev)
    out = torch.empty(n, hq, d, dtype=BF16, device=dev)
    plan.attend8(out, q.to(dev), kc.to(dev), vc.to(dev), powers.to(dev), table.to(dev), weights=w)
    torch.cuda.synchronize()
    for b in (0, 117, 199):
        want, weights, bound, w_bound = reference(q[b:b + 1], k, v, table[b:b + 1], [0], [1], [length], page, 0, d ** -0.5)
        check_out(out[b:b + 1], want, bound)
        assert bool(((w[b].cpu().double() - weights[0, :length]).abs() <= w_bound[0, :length] + 2.0 ** -22).all())
    assert float((w.sum(1) - hq).abs().max()) <= 1e-3 * hq


def test_captured_with_room_that_nobody_uses(dev):
    """Heads of 128, a list that is cut and one that is not: in one graph, replayed between eager calls, against the eager results."""
    cases = [coded(dev, 2, F16, 4, 2, 128, [(1, 900), (1, 33)], seed=14), coded(dev, 2, F16, 16, 16, 128, [(1, 1 + i) for i in range(66)], seed=15)]
    calls = []
    for c in cases:
        hq, d, hkv = c["q"].shape[1], c["q"].shape[2], c["kb"].shape[1]
        plan = AttentionPlan(*c["lengths"], n_tokens=c["T"], max_seq_len=1, max_kv_len=max(c["lens"]), q_heads=hq, kv_heads=hkv, head_dim=d,
                             page_size=2, window=0)
        args = [c[n].to(dev) for n in ("q", "key_codes", "value_codes", "powers", "table")]
        calls.append((plan, torch.zeros_like(args[0]), args))
    want = [run(dev, c, 2) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for plan, out, args in calls:
            plan.attend8(out, *args)
    for _ in range(4):
        for _, out, _ in calls:
            out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for (_, out, _), w, c in zip(calls, want, cases):
            assert torch.equal(out, w)
            assert torch.equal(run(dev, c, 2), w)
