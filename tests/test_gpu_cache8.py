"""GPU: the 8-bit cache written and read back, against its definition in 64 bits (tests/_cache8.py)."""
import math

import pytest
import torch

from tests._cache8 import decode, encode, pages_of
from valora_amd import cache8
from valora_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def rotated(x, positions, freqs, R, interleaved, gain=1.0):
    """``x`` ``[T, heads, d]`` in 64 bits; ``freqs`` in turns."""
    x = x.double().clone()
    turns = positions.double()[:, None] * freqs[None]
    angle = 2 * math.pi * (turns - turns.round())
    cos, sin = angle.cos()[:, None] * gain, angle.sin()[:, None] * gain
    a, b = (x[..., 0:R:2].clone(), x[..., 1:R:2].clone()) if interleaved else (x[..., :R // 2].clone(), x[..., R // 2:R].clone())
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        x[..., 0:R:2], x[..., 1:R:2] = ra, rb
    else:
        x[..., :R // 2], x[..., R // 2:R] = ra, rb
    return x


def empty(dev, pages, heads, page, d):
    codes = lambda: torch.full((pages, heads, page, d), 0x55, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)  # noqa: E731
    return codes(), codes(), torch.full((pages, heads, page, 2), 0x77, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)


def check_stored(kc, vc, powers, loc, k, v, dtype, page):
    """The slots hold the codes of k and v (in 64 bits, on the CPU), all others what they held.  A code may be the neighbour where k lies
    within 2^-40 of the border (the tests' sines are a device's); its sign does not matter at 0."""
    n_slots, heads, d = kc.shape[0] * page, kc.shape[1], kc.shape[3]
    ok = (loc >= 0) & (loc < n_slots)
    rows = lambda t: t.cpu().view(torch.uint8).transpose(1, 2).reshape(n_slots, heads, -1)  # noqa: E731
    got_k, got_v, got_e = rows(kc), rows(vc), rows(powers)
    for got, which, x in ((got_k, 0, k), (got_v, 1, v)):
        codes, e = encode(x[ok], dtype)
        at = loc[ok]
        assert torch.equal(got_e[at][..., which], e), "powers"
        mine = got[at]
        same = (mine == codes) | ((mine & 127 == 0) & (codes & 127 == 0)) | ((mine & 127 == 127) & (codes & 127 == 127))
        for t, h, i in torch.nonzero(~same).tolist():
            scaled = float(x[ok][t, h, i]) * 2.0 ** (127 - int(e[t, h]))
            pair = decode(torch.tensor([int(mine[t, h, i]), int(codes[t, h, i])], dtype=torch.uint8), torch.full((), 127, dtype=torch.uint8))
            assert abs(scaled - float(pair.mean())) <= 2.0 ** -40 * abs(scaled), (t, h, i, scaled, pair)
    other = torch.ones(n_slots, dtype=torch.bool)
    other[loc[ok]] = False
    assert bool((got_k[other] == 0x55).all()) and bool((got_v[other] == 0x55).all()) and bool((got_e[other] == 0x77).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,R,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (64, 32, True), (32, 32, False), (96, 96, False),
                                             (96, 48, True), (256, 256, False), (256, 64, True), (64, 22, False), (32, 6, True), (128, 2, False)])
@pytest.mark.parametrize("T,hq,hk,page", [(1, 4, 4, 2), (7, 6, 2, 1), (65, 3, 1, 16), (600, 8, 5, 4)])
def test_store_and_read(dev, dtype, d, R, interleaved, T, hq, hk, page):
    g = torch.Generator().manual_seed(T * 7 + d + R)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hk, hk))
    k[:, :, ::13] *= 30
    positions = torch.randint(0, 1 << 20, (T,), generator=g)
    pages = -(-(T + 9) // page)
    loc = torch.randperm(pages * page, generator=g)[:T]
    if T > 6:
        loc[2], loc[5], loc[6] = -1, pages * page, -(1 << 40)
    rotary = Rotary(d, rotary_dim=R, interleaved=interleaved, device=dev)
    kc, vc, powers = empty(dev, pages, hk, page, d)
    q_out = torch.full_like(q, 9.0).to(dev)
    qd, kd, vd = q.to(dev), k.to(dev), v.to(dev)
    rotary.store8(positions.to(dev), qd, kd, vd, kc, vc, powers, loc.to(dev), q_out=q_out)
    torch.cuda.synchronize()
    assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    freqs = rotary.freqs.cpu()
    k64 = rotated(k, positions, freqs, R, interleaved)
    check_stored(kc, vc, powers, loc, k64, v.double(), dtype, page)
    # q: the angle and each product in 32 bits (2^-21 of the pair's size in all), one rounding
    want = rotated(q, positions, freqs, R, interleaved)
    size = q.double().abs().amax(-1, keepdim=True)
    assert bool(((q_out.cpu().double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + size * 2.0 ** -20).all())
    # reading back gives the codes' values, whichever wrote them
    rk, rv = cache8.read(kc, vc, powers, loc.to(dev), dtype=dtype)
    rows = lambda t: t.cpu().view(torch.uint8).transpose(1, 2).reshape(pages * page, hk, -1)  # noqa: E731
    ok = (loc >= 0) & (loc < pages * page)
    for got, codes, which in ((rk, kc, 0), (rv, vc, 1)):
        want = torch.zeros(T, hk, d, dtype=torch.float64)
        want[ok] = decode(rows(codes)[loc[ok]], rows(powers)[loc[ok]][..., which])
        assert torch.equal(got.cpu().double(), want)
    # in place of q
    rotary.store8(positions.to(dev), qd, kd, vd, kc, vc, powers, loc.to(dev))
    assert torch.equal(qd, q_out)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_at_the_borders(dev, dtype):
    """Halfway between codes, at the ends of a power, zeros, subnormal ones, the type's largest, infinities and no numbers: v is stored as it
    is, k at position 0 as well."""
    d, cases = 32, []
    for top in (448.0, 449.0, 447.0, 1.75, 1.7578125, 464.0, 2.0 ** -14, float(torch.finfo(dtype).max), float(torch.finfo(dtype).tiny), 0.0):
        for at in range(4):
            x = torch.linspace(-1.0, 1.0, d, dtype=torch.float64) * top
            x[0] = top
            cases.append(x)
    grid = (torch.arange(d, dtype=torch.float64) + 0.5) / 64 + 1.0           # halves and quarters of e4m3's steps
    cases += [grid, grid * 2.0 ** -7, torch.cat([grid[:31], torch.tensor([448.0]).double()])]
    x = torch.stack(cases).to(dtype)[:, None].repeat(1, 2, 1)
    x[5, 0, 3], x[6, 0, 4], x[7, 1, :], x[8, 0, 5] = math.inf, -math.inf, math.nan, math.nan
    x[9, 1, :] = math.inf
    T = x.shape[0]
    rotary = Rotary(d, device=dev)
    kc, vc, powers = empty(dev, T, 2, 1, d)
    loc = torch.arange(T)
    k = x.clone()
    k[5:10] = 1.0                                                            # (a rotated infinity is no number in its pair)
    rotary.store8(torch.zeros(T, dtype=torch.long, device=dev), torch.zeros(T, 2, d, dtype=dtype, device=dev), k.to(dev), x.to(dev), kc, vc,
                  powers, loc.to(dev))
    check_stored(kc, vc, powers, loc, k.double(), x.double(), dtype, 1)
    rk, rv = cache8.read(kc, vc, powers, loc.to(dev), dtype=dtype)
    fine = torch.isfinite(x)
    # half a step of e4m3, above its normal range's end by the power's least step
    e = powers.cpu().view(torch.uint8)[:, :, 0, 1].double() - 127
    step = torch.maximum(x.double().abs() * 2.0 ** -4, torch.exp2(e - 10)[..., None])
    inside = fine & (x.double().abs() <= 448.0 * torch.exp2(e)[..., None])
    assert bool(((rv.cpu().double() - x.double()).abs() <= step)[inside].all())
    assert bool(torch.isnan(rv.cpu()[torch.isnan(x)]).all()) and bool(torch.isfinite(rv.cpu()[~torch.isnan(x)]).all())


def test_a_rotated_infinity_spoils_its_pair_alone(dev):
    d = 64
    k = torch.ones(3, 1, d, dtype=BF16)
    k[1, 0, 3] = math.inf
    rotary = Rotary(d, device=dev)
    kc, vc, powers = empty(dev, 4, 1, 1, d)
    args = (torch.tensor([5, 6, 7], device=dev), torch.zeros(3, 1, d, dtype=BF16, device=dev), k.to(dev), k.to(dev), kc, vc, powers,
            torch.tensor([0, 1, 2], device=dev))
    rotary.store8(*args)
    rk, _ = cache8.read(kc, vc, powers, torch.tensor([0, 1, 2], device=dev), dtype=BF16)
    rk = rk.cpu()[:, 0]
    rest = torch.ones(d, dtype=torch.bool)
    rest[3] = rest[35] = False
    want = rotated(k, torch.tensor([5, 6, 7]), rotary.freqs.cpu(), d, False)[:, 0]
    assert bool((rk[1, rest].double() - want[1, rest]).abs().max() <= 2.0 ** -4 * 2)
    assert torch.isfinite(rk[0]).all() and torch.isfinite(rk[2]).all()


def test_scaled_rotation(dev):
    """A yarn scaling's gain is part of the rotation."""
    g = torch.Generator().manual_seed(3)
    T, d = 33, 64
    k = torch.randn(T, 2, d, generator=g).to(F16)
    rotary = Rotary(d, base=500000.0, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096}, device=dev)
    positions = torch.randint(0, 16000, (T,), generator=g)
    kc, vc, powers = empty(dev, 20, 2, 2, d)
    loc = torch.randperm(40, generator=g)[:T]
    rotary.store8(positions.to(dev), k.to(dev), k.to(dev), k.to(dev), kc, vc, powers, loc.to(dev), q_out=torch.empty_like(k, device=dev))
    gain = torch.tensor(rotary.gain, dtype=torch.float32).double()
    check_stored(kc, vc, powers, loc, rotated(k, positions, rotary.freqs.cpu(), d, False, gain), k.double(), F16, 2)


def test_strides(dev):
    """One projection's output cut in three, with heads apart in k; keys' and values' pages side by side; nothing aligned to 16 bytes in v."""
    g = torch.Generator().manual_seed(4)
    T, hq, hk, d, page = 21, 4, 2, 64, 4
    qkv = torch.randn(T, hq * d + hk * (d + 8) + hk * d + 1, generator=g).to(BF16).to(dev)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:hq * d + hk * (d + 8)].unflatten(1, (hk, d + 8))[..., :d]
    v = qkv[:, hq * d + hk * (d + 8) + 1:].unflatten(1, (hk, d))
    both = torch.full((8, 2, hk, page, d), 0x55, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    powers = torch.full((8, hk, page, 2), 0x77, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
    positions, loc = torch.arange(T) * 37, torch.randperm(32, generator=g)[:T]
    rotary = Rotary(d, device=dev)
    out = torch.empty(T, hq, d + 2, dtype=BF16, device=dev)
    rotary.store8(positions.to(dev), q, k, v, both[:, 0], both[:, 1], powers, loc.to(dev), q_out=out[..., :d])
    k64 = rotated(k.cpu(), positions, rotary.freqs.cpu(), d, False)
    check_stored(both[:, 0], both[:, 1], powers, loc, k64, v.cpu().double(), BF16, page)
    k_out, v_out = torch.full((T, hk * d + 8), 3.0, dtype=BF16, device=dev), torch.full((T, hk, d), 3.0, dtype=BF16, device=dev)
    got = cache8.read(both[:, 0], both[:, 1], powers, loc.to(dev), BF16, k_out[:, :hk * d], v_out)
    dense = cache8.read(both[:, 0], both[:, 1], powers, loc.to(dev), BF16)
    assert torch.equal(got[0].reshape(T, hk, d), dense[0]) and torch.equal(v_out, dense[1]) and bool((k_out[:, hk * d:] == 3.0).all())


def test_slots_beyond_32_bits_of_bytes(dev):
    """A cache whose codes pass 2^32 bytes, at its ends."""
    hk, page, d = 8, 2, 256
    pages = (1 << 32) // (hk * page * d) + 3
    kc = torch.empty(pages, hk, page, d, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    vc = torch.empty(pages, hk, page, d, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    powers = torch.empty(pages, hk, page, 2, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, hk, d, generator=g).to(BF16)
    loc = torch.tensor([0, 2 * pages - 1, pages, 2 * pages - 2], device=dev)
    rotary = Rotary(d, device=dev)
    rotary.store8(torch.zeros(4, dtype=torch.long, device=dev), x.to(dev), x.to(dev), x.to(dev), kc, vc, powers, loc)
    k, v = cache8.read(kc, vc, powers, loc, dtype=BF16)
    codes, e = encode(x, BF16)
    want = decode(codes, e)
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), want)


def test_codes_of_rows_is_the_same_memory(dev):
    rows = torch.zeros(5, 2, 64, dtype=F16, device=dev)
    codes = cache8.codes_of_rows(rows)
    assert codes.shape == (5, 2, 2, 64) and codes.data_ptr() == rows.data_ptr()
    codes.view(torch.uint8)[3, 1, 1, 63] = 0x3c
    assert float(rows[3, 1, 63]) == 1.0
    with pytest.raises(RuntimeError, match="16-bit rows"):
        cache8.codes_of_rows(rows.float())


def test_nothing_to_do(dev):
    rotary = Rotary(64, device=dev)
    kc, vc, powers = empty(dev, 2, 1, 2, 64)
    none = torch.empty(0, 1, 64, dtype=BF16, device=dev)
    rotary.store8(torch.empty(0, dtype=torch.long, device=dev), none, none, none, kc, vc, powers, torch.empty(0, dtype=torch.long, device=dev))
    k, v = cache8.read(kc, vc, powers, torch.empty(0, dtype=torch.long, device=dev), dtype=BF16)
    assert k.shape == v.shape == (0, 1, 64)
