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


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,hq,hk,d,R,interleaved", [(6001, 4, 4, 128, 128, False), (14002, 3, 1, 64, 32, False), (2103, 8, 8, 256, 256, True),
                                                     (1301, 40, 8, 96, 96, False), (27001, 1, 2, 32, 32, True), (53002, 1, 2, 32, 32, False)])
def test_many_tokens(dev, dtype, T, hq, hk, d, R, interleaved):
    """Several tokens a workgroup, the last one's not all there; codes against those of the same tokens in small calls."""
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype).to(dev) for h in (hq, hk, hk))
    positions = torch.randint(0, 1 << 18, (T,), generator=g).to(dev)
    page = 16
    pages = T // page + 3
    loc = torch.randperm(pages * page, generator=g)[:T].to(dev)
    loc[T - 2] = -1
    rotary = Rotary(d, rotary_dim=R, interleaved=interleaved, device=dev)
    whole, parts = empty(dev, pages, hk, page, d), empty(dev, pages, hk, page, d)
    out, out_parts = torch.empty_like(q), torch.empty_like(q)
    rotary.store8(positions, q, k, v, *whole, loc, q_out=out)
    step = 40 if T < 10000 else 400
    for at in range(0, T, step):
        some = slice(at, at + step)
        rotary.store8(positions[some], q[some], k[some], v[some], *parts, loc[some], q_out=out_parts[some])
    assert torch.equal(out, out_parts)
    for a, b in zip(whole, parts):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    few = slice(T - 40, T)
    k64 = rotated(k.cpu(), positions.cpu(), rotary.freqs.cpu(), R, interleaved)
    kc, vc, powers = empty(dev, pages, hk, page, d)
    rotary.store8(positions[few], q[few], k[few], v[few], kc, vc, powers, loc[few])
    check_stored(kc, vc, powers, loc[few].cpu(), k64[few], v[few].cpu().double(), dtype, page)


def test_without_q(dev):
    """The C entry takes k and v alone."""
    import ctypes
    from valora_amd import _lib
    g = torch.Generator().manual_seed(8)
    T, hk, d, page = 13, 3, 64, 2
    k, v = (torch.randn(T, hk, d, generator=g).to(F16).to(dev) for _ in range(2))
    positions, loc = torch.arange(T, device=dev) * 11, torch.randperm(20, generator=g)[:T].to(dev)
    rotary = Rotary(d, device=dev)
    want, got = empty(dev, 10, hk, page, d), empty(dev, 10, hk, page, d)
    rotary.store8(positions, torch.zeros(T, 1, d, dtype=F16, device=dev), k, v, *want, loc)
    cache = _lib.Cache8(got[0].data_ptr(), got[1].data_ptr(), got[2].data_ptr(), 10, hk * page * d, hk * page * d, hk * page * 2, hk, d, page)
    _lib.check(_lib.lib().mlora_rotary_store_codes(_lib.current_stream(dev), None, _lib.ptr(k), hk * d, d, _lib.ptr(v), hk * d, d, ctypes.byref(cache),
                                                   _lib.ptr(positions), _lib.ptr(loc), T, d, 0, _lib.ptr(rotary.freqs), 1.0, 0))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals(dev):
    rotary = Rotary(64, device=dev)
    kc, vc, powers = empty(dev, 4, 2, 2, 64)
    x = torch.zeros(3, 2, 64, dtype=BF16, device=dev)
    pos, loc = torch.zeros(3, dtype=torch.long, device=dev), torch.arange(3, device=dev)
    good = dict(positions=pos, q=x.clone(), k=x, v=x, key_codes=kc, value_codes=vc, powers=powers, loc=loc)
    rotary.store8(**good)
    for kw, message in ((dict(key_codes=kc.view(torch.uint8)), "key_codes"), (dict(powers=powers.view(torch.uint8)), "powers"),
                        (dict(powers=powers[:3]), "powers must be"), (dict(value_codes=vc[:3]), "same shape"), (dict(value_codes=kc), "overlap"),
                        (dict(key_codes=kc.transpose(1, 2)), "contiguous"), (dict(key_codes=kc[0]), "must be"), (dict(loc=loc.int()), "loc"),
                        (dict(loc=loc[:2]), "slot per token"), (dict(k=x[:, :1]), "heads"), (dict(k=x[:2]), "row per position"),
                        (dict(v=x.half()), "No suitable kernel"), (dict(q=x.float()), "No suitable kernel"), (dict(positions=pos[:2]), "tokens"),
                        (dict(k=x.cpu()), "CUDA tensor"), (dict(powers=powers.cpu()), "CUDA tensor"), (dict(loc=loc.cpu()), "CUDA tensor")):
        with pytest.raises(RuntimeError, match=message):
            rotary.store8(**dict(good, **kw))
    with pytest.raises(RuntimeError, match="head_dim=32"):
        rotary.store8(**dict(good, key_codes=kc[..., :32].contiguous(), value_codes=vc[..., :32].contiguous()))
    for kw, message in ((dict(dtype=torch.float32), "No suitable kernel"), (dict(loc=loc.int()), "loc"), (dict(k_out=x[:2]), "row per slot"),
                        (dict(k_out=x.half()), "k_out"), (dict(k_out=x[..., ::2]), "k_out"), (dict(k_out=x, v_out=x), "k_out must not be v_out")):
        with pytest.raises(RuntimeError, match=message):
            cache8.read(**dict(dict(key_codes=kc, value_codes=vc, powers=powers, loc=loc, dtype=BF16), **kw))
    from valora_amd.attention import AttentionPlan
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    plan = AttentionPlan(i32([0]), i32([3]), i32([3]), n_tokens=3, max_seq_len=3, max_kv_len=3, q_heads=2, kv_heads=2, head_dim=64, page_size=2)
    out, table = torch.empty_like(x), i32([[0, 1]])
    good = dict(out=out, q=x, key_codes=kc, value_codes=vc, powers=powers, table=table)
    plan.attend8(**good)
    for kw, message in ((dict(q=x.float()), "No suitable kernel"), (dict(out=out.half()), "No suitable kernel"), (dict(out=x), "out must not be q"),
                        (dict(key_codes=kc.view(torch.uint8)), "key_codes"), (dict(table=table.long()), "table"), (dict(table=table[:, :1]), "max_kv_len"),
                        (dict(key_codes=kc[:, :1].contiguous(), value_codes=vc[:, :1].contiguous(), powers=powers[:, :1].contiguous()), "2 of 64 in pages of 2"),
                        (dict(weights=torch.zeros(1, 2, device=dev)), "max_kv_len"), (dict(scale=-1.0), "positive")):
        with pytest.raises(RuntimeError, match=message):
            plan.attend8(**dict(good, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_any_codes_and_powers(dev, dtype):
    """Every code, with powers that the type does not hold all values of: rounded to the nearest, infinite beyond."""
    g = torch.Generator().manual_seed(9)
    n, d = 3000, 32
    codes = torch.randint(0, 256, (n, 1, 1, d), generator=g, dtype=torch.int16).to(torch.uint8)
    powers = torch.randint(127 - 40, 127 + 20, (n, 1, 1, 2), generator=g).to(torch.uint8)
    powers[:20] = 255
    on = lambda t, f: t.to(dev).view(f)  # noqa: E731
    k, v = cache8.read(on(codes, torch.float8_e4m3fn), on(codes.flip(0), torch.float8_e4m3fn), on(powers, torch.float8_e8m0fnu), torch.arange(n, device=dev), dtype)
    for got, c, which in ((k, codes, 0), (v, codes.flip(0), 1)):
        want = decode(c[:, 0], powers[:, 0, :, which]).to(dtype)
        got = got.cpu().view_as(want)
        assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())
