"""The 8-bit cache from its definition, in 64 bits on the CPU: codes and powers of values, values of codes and powers."""
import torch

LOWEST = {torch.float16: -15, torch.bfloat16: -117}
HIGHEST = {torch.float16: 7, torch.bfloat16: 119}
# 0, the seven below 2^-6, then eight a power up to 448; a code's low seven bits are its place
GRID = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (k - 10) for k in range(1, 16) for m in range(8)], dtype=torch.float64)[:127]


def encode(x, dtype):
    """``x`` ``[..., d]``: (codes uint8 ``[..., d]``, power bytes ``[...]``)."""
    x = x.double()
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    powers = torch.tensor([2.0 ** e for e in range(LOWEST[dtype], HIGHEST[dtype] + 1)], dtype=torch.float64)
    which = torch.searchsorted(powers * 448.0, size).clamp(max=len(powers) - 1)
    y = torch.nan_to_num(x.abs() / powers[which][..., None], nan=0.0, posinf=448.0).clamp(max=448.0)
    hi = torch.searchsorted(GRID, y.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = GRID[hi] - y, y - GRID[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(torch.isnan(x), torch.full_like(code, 127), code) + 128 * (torch.signbit(x) & ~torch.isnan(x))
    return code.to(torch.uint8), (which + LOWEST[dtype] + 127).to(torch.uint8)


def decode(codes, powers):
    """In 64 bits; no number for the codes 127 and 255 and for the power 255."""
    codes = codes.view(torch.uint8).long()
    grid = torch.cat([GRID, torch.tensor([float("nan")], dtype=torch.float64)])
    v = torch.where(codes >= 128, -1.0, 1.0) * grid[codes & 127]
    two = torch.tensor([2.0 ** (e - 127) for e in range(255)] + [float("nan")], dtype=torch.float64)
    return v * two[powers.view(torch.uint8).long()][..., None]


def pages_of(rows, page):
    """``[slots, heads, ...]`` as pages ``[pages, heads, page, ...]``."""
    n = rows.shape[0] // page
    return rows[:n * page].reshape(n, page, *rows.shape[1:]).transpose(1, 2).contiguous()


def cache_of(kb, vb, page, dtype):
    """Codes and powers of caches ``[slots, heads, d]``: (key_codes, value_codes, powers, values of the keys, of the values), the values as
    ``dtype`` ``[slots, heads, d]``."""
    (kc, ke), (vc, ve) = encode(kb, dtype), encode(vb, dtype)
    powers = pages_of(torch.stack([ke, ve], -1), page).view(torch.float8_e8m0fnu)
    return (pages_of(kc, page).view(torch.float8_e4m3fn), pages_of(vc, page).view(torch.float8_e4m3fn), powers,
            decode(kc, ke).to(dtype), decode(vc, ve).to(dtype))
