"""GPU: rotary positions, in place, out of place and into the cache's rows, against the definition in 64 bits."""
import math

import pytest
import torch

from valora_amd.rotary import Rotary, frequencies

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALINGS = [None, dict(type="linear", factor=8.0), dict(type="ntk", factor=4.0),
            dict(type="bands", factor=8.0, low=1.0, high=4.0, original_max_position=8192),
            dict(type="yarn", factor=16.0, original_max_position=4096)]


def turned(x, positions, radians, gain, rotary_dim, interleaved):
    """([T, heads, d] rotated in 64 bits, how far a result may be off)"""
    x = x.detach().cpu().double()
    angle = positions.cpu().double()[:, None] * torch.tensor(radians, dtype=torch.float64)[None]
    cos, sin = (angle.cos() * gain)[:, None], (angle.sin() * gain)[:, None]
    out = x.clone()
    i = torch.arange(rotary_dim // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., a] * sin + x[..., b] * cos
    # sine and cosine: the reference's angle is rounded in 64 bits, the kernel's to 2^-25 turns and a few steps of 32 bits after
    off = angle.abs() * 2.0 ** -51 + 2 * math.pi * 2.0 ** -25 + 2.0 ** -21
    size = torch.zeros_like(x)
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * off[:, None] * abs(gain)
    return out, size


def check(got, want, size):
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == F16 else 0.0       # half the least step of fp16
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= want.abs() * u * 1.01 + size * 1.01 + tiny).all()), float((err - want.abs() * u - size).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary_dim", [(128, 128), (128, 64), (64, 64), (96, 32), (80, 20), (256, 256), (64, 2), (6, 4), (32, 30)])
@pytest.mark.parametrize("T", [1, 3, 77, 600])
def test_in_place_and_out_of_place(dev, dtype, interleaved, d, rotary_dim, T):
    g = torch.Generator().manual_seed(T + d)
    q, k = torch.randn(T, 5, d, generator=g).to(dtype), torch.randn(T, 2, d, generator=g).to(dtype)
    positions = torch.randint(0, 5000, (T,), generator=g)
    rot = Rotary(d, rotary_dim=rotary_dim, interleaved=interleaved, device=dev)
    radians, gain = frequencies(rotary_dim)
    qd, kd, pd = q.to(dev), k.to(dev), positions.to(dev)
    qo, ko = torch.full_like(qd, 9.0), torch.full_like(kd, 9.0)
    rot.apply(pd, qd, kd, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
    check(qo, *turned(q, positions, radians, gain, rotary_dim, interleaved))
    check(ko, *turned(k, positions, radians, gain, rotary_dim, interleaved))
    assert torch.equal(qo[..., rotary_dim:].cpu(), q[..., rotary_dim:])
    rot.apply(pd, qd, kd)
    torch.cuda.synchronize()
    assert torch.equal(qd, qo) and torch.equal(kd, ko)
    alone = q.to(dev).view(T, -1)                        # heads side by side in one dimension
    rot.apply(pd, alone)
    assert torch.equal(alone.view_as(qo), qo)


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_scaled_and_far_positions(dev, scaling, base):
    T, d = 64, 128
    g = torch.Generator().manual_seed(3)
    q = torch.randn(T, 2, d, generator=g).to(F16)
    positions = torch.cat([torch.arange(16), 2 ** torch.arange(12, 28), torch.randint(0, 10**6, (16,), generator=g),
                           -torch.randint(0, 10**5, (16,), generator=g)])
    rot = Rotary(d, base=base, scaling=scaling, device=dev)
    out = torch.empty_like(q, device=dev)
    rot.apply(positions.to(dev), q.to(dev), q_out=out)
    radians, gain = frequencies(d, base, scaling)
    check(out, *turned(q, positions, radians, gain, d, False))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,rotary_dim,interleaved", [(32, 8, 128, 128, False), (4, 4, 64, 32, True), (3, 1, 80, 20, False), (7, 1, 96, 96, True)])
@pytest.mark.parametrize("T", [1, 33, 700])
def test_store(dev, dtype, hq, hkv, d, rotary_dim, interleaved, T):
    """q, k, v are slices of one projection's output, the buffers' rows are apart; rows outside the pool are not written."""
    g = torch.Generator().manual_seed(T)
    fused = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(dtype)
    q, k, v = (t.unflatten(1, (-1, d)) for t in fused.split([hq * d, hkv * d, hkv * d], 1))
    positions = torch.randint(0, 100000, (T,), generator=g)
    rows = T + 9
    loc = torch.randperm(rows, generator=g)[:T]
    if T > 2:
        loc[1], loc[2] = -1, rows
    rot = Rotary(d, rotary_dim=rotary_dim, interleaved=interleaved, device=dev)
    fd = fused.to(dev)
    qd, kd, vd = (t.unflatten(1, (-1, d)) for t in fd.split([hq * d, hkv * d, hkv * d], 1))
    pool = torch.full((rows, 2, hkv + 1, d), 5.0, dtype=dtype, device=dev)
    kb, vb = pool[:, 0, :hkv], pool[:, 1, 1:]
    out = torch.empty(T, hq, d, dtype=dtype, device=dev)
    rot.store(positions.to(dev), qd, kd, vd, kb, vb, loc.to(dev), q_out=out)
    torch.cuda.synchronize()
    assert torch.equal(fd.cpu(), fused)
    radians, gain = frequencies(rotary_dim)
    check(out, *turned(q, positions, radians, gain, rotary_dim, interleaved))
    want, size = turned(k, positions, radians, gain, rotary_dim, interleaved)
    there = (loc >= 0) & (loc < rows)
    check(kb.cpu()[loc[there]], want[there], size[there])
    assert torch.equal(vb.cpu()[loc[there]], v[there])
    touched = torch.zeros(rows, dtype=torch.bool)
    touched[loc[there]] = True
    assert bool((pool.cpu()[~touched] == 5.0).all()) and bool((pool[:, 0, hkv].cpu() == 5.0).all()) and bool((pool[:, 1, 0].cpu() == 5.0).all())
    rot.store(positions.to(dev), qd, kd, vd, kb, vb, loc.to(dev))          # q in place
    torch.cuda.synchronize()
    assert torch.equal(qd, out) and torch.equal(fd[:, hq * d:].cpu(), fused[:, hq * d:])


def test_slices_that_begin_anywhere(dev):
    """Rows and heads that are not multiples of 16 bytes apart, or begin in between."""
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(50, 3, 131, generator=g).to(F16)
    positions = torch.randint(0, 3000, (50,), generator=g)
    rot = Rotary(64, device=dev)
    for at in (0, 1, 2, 8, 67):
        wd = wide.to(dev)
        x = wd[:, :, at:at + 64]
        rot.apply(positions.to(dev), x)
        torch.cuda.synchronize()
        check(x, *turned(wide[:, :, at:at + 64], positions, *frequencies(64), 64, False))
        rest = torch.ones(131, dtype=torch.bool)
        rest[at:at + 64] = False
        assert torch.equal(wd.cpu()[:, :, rest], wide[:, :, rest])


def test_values_that_are_not_finite_stay_in_their_pair(dev):
    q = torch.ones(4, 1, 64, dtype=F16)
    q[0, 0, 3], q[1, 0, 40], q[2, 0, 60] = math.nan, math.inf, -math.inf
    rot = Rotary(64, rotary_dim=48, device=dev)
    out = q.to(dev)
    rot.apply(torch.arange(1, 5, device=dev), out)
    bad = ~torch.isfinite(out[:, 0].cpu())
    assert sorted(bad.nonzero().tolist()) == [[0, 3], [0, 27], [1, 16], [1, 40], [2, 60]]


def test_replayed_graph_and_another_stream(dev):
    T, d = 40, 128
    g = torch.Generator().manual_seed(5)
    rot = Rotary(d, device=dev)
    q, k, v = (torch.randn(T, 4, d, generator=g).to(BF16).to(dev) for _ in range(3))
    pos, loc = torch.arange(T, device=dev), torch.arange(T, device=dev)
    kb, vb, out = (torch.zeros(T, 4, d, dtype=BF16, device=dev) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rot.store(pos, q, k, v, kb, vb, loc, q_out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.store(pos, q, k, v, kb, vb, loc, q_out=out)
    for step in range(3):
        pos.add_(1000)
        loc.copy_(torch.randperm(T, generator=g))
        kb.zero_(), vb.zero_(), out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        k2, v2, o2 = torch.zeros_like(kb), torch.zeros_like(vb), torch.zeros_like(out)
        rot.store(pos, q, k, v, k2, v2, loc, q_out=o2)
        torch.cuda.synchronize()
        assert torch.equal(k2, kb) and torch.equal(v2, vb) and torch.equal(o2, out) and bool(out.any())


def test_no_tokens(dev):
    rot = Rotary(64, device=dev)
    e = torch.empty(0, 2, 64, dtype=F16, device=dev)
    i = torch.empty(0, dtype=torch.long, device=dev)
    rot.apply(i, e)
    rot.store(i, e, e, e, torch.zeros(3, 2, 64, dtype=F16, device=dev), torch.zeros(3, 2, 64, dtype=F16, device=dev), i)


def test_refusals(dev):
    rot = Rotary(64, device=dev)
    x = torch.zeros(3, 2, 64, dtype=F16, device=dev)
    p = torch.zeros(3, dtype=torch.long, device=dev)
    pool = torch.zeros(8, 2, 64, dtype=F16, device=dev)
    cases = [(lambda: rot.apply(p.int(), x), "scalar type Long"), (lambda: rot.apply(p.cpu(), x), "CUDA"), (lambda: rot.apply(p, x.cpu()), "CUDA"),
             (lambda: rot.apply(p[:2], x), "tokens"), (lambda: rot.apply(p, x.float()), "No suitable kernel"),
             (lambda: rot.apply(p, x, x.bfloat16()), "No suitable kernel"), (lambda: rot.apply(p, x[..., :32]), "must be"),
             (lambda: rot.apply(p, x.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
             (lambda: rot.apply(p, x, q_out=x[:, :1]), "differ"), (lambda: rot.apply(p, x, k_out=x), "k_out"),
             (lambda: rot.store(p, x, x, x, pool, pool[:4], p), "same rows"), (lambda: rot.store(p, x, x, x, pool, pool, p.int()), "Long"),
             (lambda: rot.store(p, x, x, x, pool, pool, p[:2]), "loc"), (lambda: rot.store(p, x, x, x, pool[:, :1], pool, p), "differ"),
             (lambda: rot.store(p, x, x, x, pool.bfloat16(), pool, p), "No suitable kernel")]
    for call, message in cases:
        with pytest.raises(RuntimeError, match=message):
            call()
