"""GPU: attention over the paged cache against the definition in 64 bits, at the lengths, head layouts, pages and masks where
tiles, pieces and lists begin and end."""
import math

import pytest
import torch

from tests._attention import attend as reference, check_out
from valora_amd.attention import AttentionPlan

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(dev, dtype, hq, hkv, d, page, reqs, seed=0, gap=0, sharp=1.0, spare=3, fill=None):
    """Requests [(new, cached)] with their rows of q ``gap`` apart and their pages scattered over the pool."""
    g = torch.Generator().manual_seed(seed)
    starts, at = [], gap
    for n, _ in reqs:
        starts.append(at)
        at += n + gap
    T = at
    counts = [-(-l // page) for _, l in reqs]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(reqs), max(counts + [1]) + 1), -1, dtype=torch.int32)
    o = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[o:o + c]
        o += c
    q = (torch.randn(T, hq, d, generator=g) * sharp).to(dtype)
    kb, vb = torch.randn(total * page, hkv, d, generator=g).to(dtype), torch.randn(total * page, hkv, d, generator=g).to(dtype)
    if fill is not None:      # everything in the pool that no request's token owns
        owned = torch.zeros(total * page, dtype=torch.bool)
        for b, (_, l) in enumerate(reqs):
            j = torch.arange(l)
            owned[table[b].long()[j // page] * page + j % page] = True
        kb[~owned], vb[~owned] = fill, fill
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(q=q, kb=kb, vb=vb, table=table, starts=starts, news=[n for n, _ in reqs], lens=[l for _, l in reqs], T=T,
                lengths=(i32(starts), i32([n for n, _ in reqs]), i32([l for _, l in reqs])))


def run(dev, c, page, window=0, scale=None, weights=None, out=None, max_seq=None, max_kv=None, plan=None):
    hq, d, hkv = c["q"].shape[1], c["q"].shape[2], c["kb"].shape[1]
    if plan is None:
        plan = AttentionPlan(*c["lengths"], n_tokens=c["T"], max_seq_len=max(c["news"] + [0]) if max_seq is None else max_seq,
                             max_kv_len=max(c["lens"] + [0]) if max_kv is None else max_kv, q_heads=hq, kv_heads=hkv, head_dim=d,
                             page_size=page, window=window)
    if out is None:
        out = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device=dev)
    plan.attend(out, c["q"].to(dev), c["kb"].to(dev), c["vb"].to(dev), c["table"].to(dev), scale=scale, weights=weights)
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


LONG = [(1, 1), (1, 31), (1, 32), (1, 33), (1, 129), (1, 255), (1, 257), (1, 700)]
MIXED = [(1, 300), (0, 40), (5, 5), (17, 17), (16, 100), (128, 128), (129, 200), (1, 1), (70, 1000), (2, 66)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (28, 4, 64), (6, 2, 96), (4, 4, 32), (2, 1, 256), (16, 1, 256)])
@pytest.mark.parametrize("page", [1, 16])
def test_heads_and_lengths(dev, dtype, hq, hkv, d, page):
    check(dev, make(dev, dtype, hq, hkv, d, page, LONG, seed=1, gap=1), page)
    check(dev, make(dev, dtype, hq, hkv, d, page, MIXED, seed=2, gap=2), page)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 260])
def test_new_tokens_around_the_tiles(dev, n):
    """Every number of rows at which a list, a wave or a tile begins, with the cached length at and around multiples of a tile."""
    check(dev, make(dev, BF16, 4, 1, 64, 1, [(n, n), (n, n + 63), (n, n + 64), (n, n + 65), (n, n + 511)], seed=n), 1)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 128, 256])
def test_pages_that_end_inside_a_tile(dev, page):
    check(dev, make(dev, F16, 4, 2, 64, page, [(1, 77), (3, 130), (40, 300), (1, 256), (1, 257)], seed=page, fill=math.nan), page)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
def test_window(dev, window):
    reqs = [(1, 1), (1, 64), (1, 777), (5, 300), (90, 90), (130, 900), (16, 16)]
    check(dev, make(dev, BF16, 8, 4, 64, 1, reqs, seed=window), 1, window)
    check(dev, make(dev, F16, 4, 4, 128, 16, reqs, seed=window + 1), 16, window)


@pytest.mark.parametrize("pieces", [(1, 20000, 1, 1), (40, 9000, 1, 1), (1, 5000, 4, 1), (300, 8200, 8, 1)])
def test_long_caches_in_many_pieces(dev, pieces):
    """One request alone is cut into as many pieces as the lists allow."""
    n, length, hq, hkv = pieces
    check(dev, make(dev, BF16, hq, hkv, 64, 1, [(n, length)], seed=3, sharp=2.0), 1)


def test_rows_that_see_nothing_become_zeros(dev):
    # more new tokens than cached ones: the first rows lie before the cache's first token; an empty cache; a window
    c = make(dev, F16, 4, 2, 64, 1, [(5, 2), (3, 0), (40, 7), (1, 0), (200, 100)], seed=4)
    got, _, _ = check(dev, c, 1)
    for b, (n, l) in enumerate(zip(c["news"], c["lens"])):
        assert not got[c["starts"][b]:c["starts"][b] + n - l].any()
    check(dev, c, 1, window=3)
    check(dev, make(dev, BF16, 1, 1, 128, 16, [(0, 0), (2, 0)], seed=5), 16)


def test_pages_outside_the_pool_are_seen_by_no_one(dev):
    for n_new in (1, 50):
        c = make(dev, BF16, 4, 2, 64, 16, [(n_new, 200), (n_new, 90), (n_new, 64)], seed=6)
        c["vb"][0:16] = math.inf      # what stands in for a page that is not there must not show
        c["kb"][0:16] = math.nan
        c["table"][c["table"] == 0] = 1_000_000
        c["table"][0, 3], c["table"][0, 5] = -1, -2**31
        c["table"][1, :] = 2**31 - 1
        got, _, _ = check(dev, c, 16)
        at = c["starts"][1]
        assert not got[at:at + n_new].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,length", [(9, 40), (60, 60), (130, 400)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, "max"])
def test_what_a_row_does_not_see_does_not_show(dev, dtype, n, length, value):
    """Later tokens, tokens behind the window and the rest of the last page hold values that are not finite; rows that do see them
    follow the arithmetic."""
    value = torch.finfo(dtype).max if value == "max" else value
    for window in (0, 11):
        c = make(dev, dtype, 4, 2, 64, 16, [(n, length)], seed=7, fill=value)
        j = length - 3
        row = int(c["table"][0, j // 16]) * 16 + j % 16
        c["vb"][row, 0, 5] = value                       # one element of one token that the last three rows see
        c["vb"][row, 1, :] = value
        got, _, _ = check(dev, c, 16, window)
        assert bool(torch.isfinite(got[:n - 3].float()).all()) or value == torch.finfo(dtype).max
        first = length - n                               # and a token that only the first rows still see through the window
        row = int(c["table"][0, first // 16]) * 16 + first % 16
        c["kb"][row], c["vb"][row] = (value, value) if window else (c["kb"][row], c["vb"][row])
        if value != value and window:
            got = run(dev, c, 16, window)
            assert bool(torch.isfinite(got[window:n - 3].float()).all())


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("reqs", [[(1, 200), (2, 70)], [(100, 300)], [(100, 1300)]])
def test_an_infinity_that_every_row_sees(dev, value, reqs):
    """In tiles that no mask touches, in a request of one piece and of several: it shows in its column and nowhere else."""
    c = make(dev, F16, 2, 2, 64, 1, reqs, seed=22)
    for b in range(len(reqs)):
        c["vb"][int(c["table"][b, 5]), 0, 3] = value
    check(dev, c, 1)


def test_infinities_of_both_signs_and_scores_of_minus_infinity(dev):
    c = make(dev, BF16, 2, 2, 64, 1, [(20, 20), (40, 70)], seed=8)
    rows = c["table"][0].long()
    c["vb"][rows[3], 0, 0], c["vb"][rows[6], 0, 0], c["vb"][rows[9], 1, 1] = math.inf, -math.inf, math.inf
    check(dev, c, 1)
    # a key of infinities: scores of -infinity for the rows whose q points away, which give it no weight
    c = make(dev, F16, 1, 1, 32, 1, [(3, 3), (33, 50)], seed=9)
    c["q"][:, 0, :] = c["q"][:, 0, :].abs()
    for b in (0, 1):
        c["kb"][c["table"][b].long()[:1], 0, :] = -math.inf
        c["vb"][c["table"][b].long()[:1], 0, :] = 3.0
    got = run(dev, c, 1)
    assert bool(torch.isfinite(got.float()).all()) and not got[0].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("reqs", [[(1, 100), (5, 300), (3, 9)], [(40, 90), (150, 400)], [(1, 30), (140, 600), (2, 40)]])
def test_a_row_of_nan_stands_alone(dev, dtype, reqs):
    """q of one row a request is not a number: that row is none either, the others do not notice."""
    c = make(dev, dtype, 4, 2, 64, 1, reqs, seed=21)
    want, _, bound, _ = reference(c["q"], c["kb"], c["vb"], c["table"], c["starts"], c["news"], c["lens"], 1, 0, 64 ** -0.5)
    for at, n in zip(c["starts"], c["news"]):
        c["q"][at + n // 2, 1, 7] = math.nan
        bound[at + n // 2, 1] = math.nan
    got = run(dev, c, 1)
    check_out(got, want, bound)
    for at, n in zip(c["starts"], c["news"]):
        assert bool(torch.isnan(got[at + n // 2, 1].float()).all())


@pytest.mark.parametrize("scale", [1e-6, 0.05, 30.0])
def test_scales(dev, scale):
    check(dev, make(dev, F16, 4, 4, 64, 1, [(1, 300), (50, 80)], seed=10), 1, scale=scale)


def test_growing_scores_move_the_maximum(dev):
    """Each tile's scores are above the last one's by far more than the reference may lag behind; and below."""
    for sign in (1.0, -1.0):
        c = make(dev, F16, 2, 2, 64, 1, [(1, 600), (40, 600)], seed=11)
        ramp = torch.linspace(-4, 4, 600) * sign
        for b in (0, 1):
            c["kb"][c["table"][b].long()[:600]] = ramp[:, None, None].expand(600, 2, 64).to(F16)
        c["q"][:] = 2.0
        check(dev, c, 1)


def test_equal_scores_over_a_long_cache_average(dev):
    c = make(dev, BF16, 8, 1, 64, 1, [(1, 30000)], seed=12)
    c["q"][:] = 0
    check(dev, c, 1)


def test_strides(dev):
    """q a slice of a fused projection, out and pool rows with something between, tables and weights that are slices."""
    hq, hkv, d = 6, 2, 64
    c = make(dev, BF16, hq, hkv, d, 1, [(1, 300), (45, 90), (3, 40)], seed=13)
    want, w_want, bound, w_bound = reference(c["q"], c["kb"], c["vb"], c["table"], c["starts"], c["news"], c["lens"], 1, 0, d ** -0.5)
    T, rows = c["T"], c["kb"].shape[0]
    fused = torch.full((T, (hq + 2 * hkv) * d + 8), math.nan, dtype=BF16, device=dev)
    fused[:, 8:8 + hq * d] = c["q"].view(T, -1).to(dev)
    q = fused[:, 8:8 + hq * d]
    pool = torch.full((rows, 2 * hkv + 1, d), math.nan, dtype=BF16, device=dev)
    pool[:, :hkv], pool[:, hkv:2 * hkv] = c["kb"].to(dev), c["vb"].to(dev)
    kb, vb = pool[:, :hkv], pool[:, hkv:2 * hkv]
    out = torch.full((T, 2, hq, d), 7.0, dtype=BF16, device=dev)
    table = torch.full((3, 1000), 5, dtype=torch.int32, device=dev)
    table[:, 100:100 + c["table"].shape[1]] = c["table"].to(dev)
    w = torch.zeros(3, 900, device=dev)
    plan = AttentionPlan(*c["lengths"], n_tokens=T, max_seq_len=45, max_kv_len=300, q_heads=hq, kv_heads=hkv, head_dim=d)
    plan.attend(out[:, 1], q, kb, vb, table[:, 100:100 + c["table"].shape[1]], weights=w[:, 10:310])
    torch.cuda.synchronize()
    check_out(out[:, 1], want, bound)
    assert bool((out[:, 0] == 7.0).all())
    check_out(w[:, 10:310], w_want[:, :300], w_bound[:, :300])
    assert not w[:, :10].any() and not w[:, 310:].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,page,window", [(4, 4, 128, 1, 0), (8, 2, 64, 16, 0), (8, 1, 32, 1, 70), (2, 2, 256, 4, 0), (3, 1, 96, 1, 5)])
def test_weights(dev, dtype, hq, hkv, d, page, window):
    c = make(dev, dtype, hq, hkv, d, page, [(1, 1), (1, 255), (1, 256), (1, 600), (0, 50), (30, 64), (70, 700), (140, 140), (4, 2)], seed=14, sharp=2.0)
    before = torch.rand(9, c["table"].shape[1] * page + 3, generator=torch.Generator().manual_seed(1)).to(dev)
    w = before.clone()
    _, want, w_bound = check(dev, c, page, window, weights=w)
    got = (w - before).cpu().double()
    pad = torch.zeros(9, 3, dtype=torch.float64)
    want, w_bound = torch.cat([want, pad], 1), torch.cat([w_bound, pad], 1)
    # adding to what was there rounds once, the difference taken here is exact enough: half a step of the larger sum each
    room = (before.cpu().double() + want) * 2.0 ** -23 + w_bound
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() / room.clamp_min(1e-30)).max())
    for b, l in enumerate(c["lens"]):
        assert torch.equal(w[b, l:], before[b, l:]), "behind the cached tokens"
    # each row gives 1 in all, where it sees anything
    alone = torch.zeros(9, c["table"].shape[1] * page, device=dev)
    run(dev, c, page, window, weights=alone)
    rows = torch.tensor([hq * min(n, l) for n, l in zip(c["news"], c["lens"])], dtype=torch.float64)
    assert torch.allclose(alone.sum(1).cpu().double(), rows, rtol=1e-4, atol=1e-4)


def test_weights_where_the_scores_have_no_room(dev):
    """16 new tokens on 64 heads over 66000 cached ones: more scores than are kept, so K is read again."""
    n, length, h, d = 16, 66000, 64, 32
    g = torch.Generator(device=dev).manual_seed(21)
    q = (torch.randn(n, h, d, device=dev, generator=g) * 2).to(BF16)
    kb, vb = (torch.randn(length, h, d, device=dev, generator=g).to(BF16) for _ in range(2))
    table = torch.randperm(length, device=dev, generator=g).to(torch.int32)[None]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    plan = AttentionPlan(i32([0]), i32([n]), i32([length]), n_tokens=n, max_seq_len=n, max_kv_len=length, q_heads=h, kv_heads=h, head_dim=d)
    assert n * h * length > 1 << 26
    out, w = torch.empty_like(q), torch.zeros(1, length, device=dev)
    plan.attend(out, q, kb, vb, table, weights=w)
    rows, j = table[0].long(), torch.arange(length, device=dev)
    hidden = j[None] > torch.arange(length - n, length, device=dev)[:, None]
    want, size = torch.zeros(length, dtype=torch.float64, device=dev), torch.zeros(length, dtype=torch.float64, device=dev)
    for head in range(h):
        K, Q = kb[rows, head].double(), q[:, head].double()
        p = torch.softmax((Q @ K.T.contiguous() * d ** -0.5).masked_fill(hidden, -math.inf), -1)
        rel = (2 * d + 8) * 2.0 ** -24 * float((Q.abs() @ K.abs().T.contiguous()).max()) * d ** -0.5 + 2.0 ** -20
        want += p.sum(0)
        size += p.sum(0) * (2 * rel + (length + 64) * 2.0 ** -24)
        o = p @ vb[rows, head].double()
        assert float((out[:, head].double() - o).abs().max()) <= 2.0 ** -8 * 2.5 * float((p @ vb[rows, head].double().abs()).max())
    assert bool(((w[0].double() - want).abs() <= size + 2.0 ** -60).all())


def test_the_same_call_gives_the_same_bits(dev):
    c = make(dev, BF16, 8, 2, 128, 1, MIXED + [(1, 6000)], seed=15)
    w = [torch.zeros(len(c["lens"]), c["table"].shape[1], device=dev) for _ in range(3)]
    outs = [run(dev, c, 1, weights=x) for x in w]
    for o, x in zip(outs[1:], w[1:]):
        assert torch.equal(o, outs[0]) and torch.equal(x, w[0])


def test_order_of_requests_does_not_matter(dev):
    """The same request alone and among others gives the same numbers up to how it is cut."""
    c = make(dev, F16, 4, 2, 64, 1, [(1, 500), (33, 300), (2, 90)], seed=16)
    got = run(dev, c, 1)
    order = [2, 0, 1]
    d = dict(c, table=c["table"][order], starts=[c["starts"][i] for i in order], news=[c["news"][i] for i in order],
             lens=[c["lens"][i] for i in order], lengths=tuple(t[order].contiguous() for t in c["lengths"]))
    assert torch.equal(run(dev, d, 1), got)


def test_lengths_that_do_not_fit_are_left_out_or_cut(dev):
    reqs = [(1, 100), (6, 80), (1, 50), (2, 60)]
    c = make(dev, BF16, 4, 4, 64, 1, reqs, seed=17)
    start, new, kv = c["lengths"]
    # request 1 has more new tokens than max_seq_len; request 2 starts behind the last row; request 3 has more cached tokens than max_kv_len
    start[2], kv[3] = c["T"], 10**9
    plan = AttentionPlan(start, new, kv, n_tokens=c["T"], max_seq_len=2, max_kv_len=60, q_heads=4, kv_heads=4, head_dim=64)
    got = run(dev, c, 1, plan=plan)
    want, _, bound, _ = reference(c["q"], c["kb"], c["vb"], c["table"], [c["starts"][0], c["starts"][3]], [1, 2], [60, 60], 1, 0, 0.125)
    # (request 0 sees its first 60 tokens only)
    ref0 = reference(c["q"], c["kb"], c["vb"], c["table"], [c["starts"][0]], [1], [60], 1, 0, 0.125)
    check_out(got[:1], ref0[0][:1], ref0[2][:1])
    ref3 = reference(c["q"], c["kb"], c["vb"], c["table"][3:], [c["starts"][3]], [2], [60], 1, 0, 0.125)
    s = c["starts"][3]
    check_out(got[s:s + 2], ref3[0][s:s + 2], ref3[2][s:s + 2])
    assert bool((got[1:s] == 7.0).all())
    for bad in (-1, -2**31, 2**31 - 1):
        new2, start2, kv2 = new.clone(), start.clone(), kv.clone()
        new2[:], start2[0], kv2[1] = bad, bad, bad
        plan = AttentionPlan(start2, new2, kv2, n_tokens=c["T"], max_seq_len=2, max_kv_len=60, q_heads=4, kv_heads=4, head_dim=64)
        assert bool((run(dev, c, 1, plan=plan) == 7.0).all())


def test_nothing_to_do(dev):
    e = lambda *s, dt=BF16: torch.empty(*s, dtype=dt, device=dev)  # noqa: E731
    i = torch.empty(0, dtype=torch.int32, device=dev)
    plan = AttentionPlan(i, i, i, n_tokens=0, max_seq_len=0, max_kv_len=0, q_heads=4, kv_heads=2, head_dim=64)
    plan.attend(e(0, 4, 64), e(0, 4, 64), e(8, 2, 64), e(8, 2, 64), e(0, 0, dt=torch.int32))
    z = torch.zeros(3, dtype=torch.int32, device=dev)
    plan = AttentionPlan(z, z, z, n_tokens=5, max_seq_len=1, max_kv_len=10, q_heads=4, kv_heads=2, head_dim=64)
    out = torch.full((5, 4, 64), 7.0, dtype=BF16, device=dev)
    plan.attend(out, torch.zeros_like(out), e(8, 2, 64), e(8, 2, 64), torch.zeros(3, 10, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())


def test_decode_steps_of_one_graph(dev):
    """The plan is cut again and the attention done by a replayed graph while the lengths grow; eager work goes on between."""
    hq, hkv, d, B, cap = 8, 2, 64, 6, 900
    g = torch.Generator().manual_seed(18)
    kb, vb = (torch.randn(B * cap, hkv, d, generator=g).to(BF16) for _ in range(2))
    table = torch.randperm(B * cap, generator=g).view(B, cap).to(torch.int32)
    kd, vd, td = kb.to(dev), vb.to(dev), table.to(dev)
    kv = torch.tensor([1, 30, 255, 256, 500, 800], dtype=torch.int32, device=dev)
    start, new = torch.arange(B, dtype=torch.int32, device=dev), torch.ones(B, dtype=torch.int32, device=dev)
    q, out = torch.zeros(B, hq, d, dtype=BF16, device=dev), torch.zeros(B, hq, d, dtype=BF16, device=dev)
    w = torch.zeros(B, cap, device=dev)
    plan = AttentionPlan(start, new, kv, n_tokens=B, max_seq_len=1, max_kv_len=cap, q_heads=hq, kv_heads=hkv, head_dim=d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan.attend(out, q, kd, vd, td, weights=w)      # warm-up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.rebuild()
        plan.attend(out, q, kd, vd, td, weights=w)
    for step in range(4):
        qs = torch.randn(B, hq, d, generator=g).to(BF16)
        q.copy_(qs)
        kv.add_(17)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        lens = kv.cpu().tolist()
        want, ww, bound, wb = reference(qs, kb, vb, table, list(range(B)), [1] * B, lens, 1, 0, d ** -0.5)
        check_out(out, want, bound, f"replay {step}")
        check_out(w, ww, wb + 2.0 ** -60, f"weights of replay {step}")
        eager = AttentionPlan(start, new, kv, n_tokens=B, max_seq_len=1, max_kv_len=cap, q_heads=hq, kv_heads=hkv, head_dim=d)
        out2, w2 = torch.empty_like(out), torch.zeros_like(w)
        eager.attend(out2, q, kd, vd, td, weights=w2)
        torch.cuda.synchronize()
        assert torch.equal(out2, out) and torch.equal(w2, w)


def test_on_another_stream(dev):
    c = make(dev, F16, 4, 2, 128, 1, MIXED, seed=19)
    want = run(dev, c, 1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(dev, c, 1)
    assert torch.equal(got, want)


def test_a_pool_of_more_than_four_gigabytes(dev):
    """Byte offsets of rows beyond 32 bits, of both buffers."""
    hkv, d, rows = 32, 128, 600_000
    kb = torch.empty(rows, hkv, d, dtype=BF16, device=dev)
    vb = torch.empty(rows, hkv, d, dtype=BF16, device=dev)
    g = torch.Generator().manual_seed(20)
    lens, news = [300, 200], [1, 40]
    picked = (rows - 1 - torch.randperm(60_000, generator=g)[:500]).to(torch.int32)
    small_k, small_v = (torch.randn(500, hkv, d, generator=g).to(BF16) for _ in range(2))
    kb[picked.long().to(dev)], vb[picked.long().to(dev)] = small_k.to(dev), small_v.to(dev)
    table = torch.full((2, 300), -1, dtype=torch.int32)
    table[0], table[1, :200] = picked[:300], picked[300:]
    local = torch.full((2, 300), -1, dtype=torch.int32)
    local[0], local[1, :200] = torch.arange(300), torch.arange(300, 500)
    q = torch.randn(41, hkv, d, generator=g).to(BF16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    plan = AttentionPlan(i32([0, 1]), i32(news), i32(lens), n_tokens=41, max_seq_len=40, max_kv_len=300, q_heads=hkv, kv_heads=hkv, head_dim=d)
    out, w = torch.empty(41, hkv, d, dtype=BF16, device=dev), torch.zeros(2, 300, device=dev)
    plan.attend(out, q.to(dev), kb, vb, table.to(dev), weights=w)
    torch.cuda.synchronize()
    want, ww, bound, wb = reference(q, small_k, small_v, local, [0, 1], news, lens, 1, 0, d ** -0.5)
    check_out(out, want, bound)
    check_out(w, ww[:, :300], wb[:, :300] + 2.0 ** -60)
