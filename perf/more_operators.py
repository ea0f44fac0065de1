"""Performance cases of serving from an 8-bit cache, and of the norms around a layer's blocks.

A cached token's k or v of a key head is held as ``head_dim`` values of 8 bits (e4m3) times one power of two (e8m0, a byte): the least
power with which the head's largest element is at most 448, e4m3's largest value.  Codes lie ``[pages, kv_heads, page, head_dim]``, powers
``[pages, kv_heads, page, 2]`` (k's, v's).

* ``keep``    a layer's new tokens: q rotated, the rotated k and v written as codes, and those tokens read back
* ``read``    cached tokens read back as 16-bit values, as for a request that moves elsewhere
* ``attend``  every new token attends over its request's cached tokens (its own and later new ones masked causally), with
              ``weights`` also adding up how much attention each cached token got
* ``norm``    a block's output, normalised and gated where the model does that, joins the residual stream, and what the next block reads is
              normalised
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
POWERS = {"fp16": (-15, 7), "bf16": (-117, 119)}      # with these a code times its power is a value of the type
MAX_BYTES = 1.69e9     # no drawn case moves or computes more than the largest listed ones
MAX_FLOPS = 9.6e10


def _keep(name, dtype, **kw):
    c = {"name": name, "op": "keep", "dtype": dtype, "q_heads": 32, "kv_heads": 32, "head_dim": 128, "rotary_dim": 128,
         "interleaved": False, "page": 2, "tokens": 1, "farthest": 4096}
    c.update(kw)
    return c


def _read(name, dtype, **kw):
    c = {"name": name, "op": "read", "dtype": dtype, "kv_heads": 32, "head_dim": 128, "page": 2, "tokens": 1}
    c.update(kw)
    return c


def _attend(name, dtype, **kw):
    c = {"name": name, "op": "attend", "dtype": dtype, "q_heads": 32, "kv_heads": 32, "head_dim": 128, "page": 2, "window": 0,
         "decode": 0, "ctx_min": 1, "ctx_max": 1, "chunks": 0, "chunk_min": 1, "chunk_max": 1, "past_min": 0, "past_max": 0,
         "weights": False, "lengths": 1}
    c.update(kw)
    return c


def _norm(name, dtype, **kw):
    c = {"name": name, "op": "norm", "dtype": dtype, "kind": "rms", "tokens": 1, "width": 4096, "block": True, "post": False, "gate": "none",
         "bias": False, "residual_scale": 1.0, "block_scale": 1.0}
    c.update(kw)
    return c


def listed():
    return [
        # a lone request decoding: nothing but latency
        _keep("keep_1", "fp16"),
        # a decode batch deep in long contexts, pairs side by side, half of the head rotated, grouped heads
        _keep("keep_77_partial", "bf16", kv_heads=8, rotary_dim=64, interleaved=True, tokens=77, farthest=200000),
        # a long prompt, pages of 16 tokens
        _keep("keep_8191", "bf16", kv_heads=8, page=16, tokens=8191, farthest=16000),
        # a request of a few hundred tokens leaves
        _read("read_517", "fp16", tokens=517),
        # a long one, grouped heads
        _read("read_40001", "bf16", kv_heads=8, page=16, tokens=40001),
        # a lone request decoding over a short context: latency again
        _attend("decode_1", "fp16", decode=1, ctx_min=517, ctx_max=517),
        # the headline decode batch, contexts of a few hundred to two thousand tokens, a key head per query head
        _attend("decode_256", "fp16", decode=256, ctx_min=200, ctx_max=2000, lengths=3),
        # few requests with very long contexts, grouped heads, pages of 16 tokens
        _attend("decode_5_long", "bf16", kv_heads=8, page=16, decode=5, ctx_min=30000, ctx_max=70000, lengths=5),
        # a chunk of a long prompt over what is cached of it, among decoding requests
        _attend("chunk_500_of_12000", "bf16", kv_heads=8, page=16, decode=31, ctx_min=500, ctx_max=3500, chunks=1, chunk_min=500,
                chunk_max=500, past_min=11500, past_max=11500, lengths=9),
        # one token's residual stream: latency
        _norm("norm_1", "fp16"),
        # a decode batch of a wider model with norms before and after its blocks
        _norm("norm_256_post", "bf16", tokens=256, width=5120, post=True),
        # a long prompt, a learned gate on each channel
        _norm("norm_8191_gate", "bf16", tokens=8191, width=4096, gate="channel"),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["keep", "read", "attend", "attend", "norm"])
    heads = rng.choice([(32, 32), (32, 8), (40, 40), (16, 2), (28, 4), (8, 1)])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "keep":
        d = rng.choice([32, 64, 96, 128, 128, 256])
        c = _keep("", dtype, q_heads=heads[0], kv_heads=heads[1], head_dim=d, rotary_dim=rng.choice([d, d, d // 2]),
                  interleaved=rng.random() < 0.5, page=rng.choice([1, 2, 2, 16, 64]), tokens=between(1, 8191), farthest=between(2048, 400000))
    elif op == "read":
        c = _read("", dtype, kv_heads=heads[1], head_dim=rng.choice([32, 64, 96, 128, 128, 256]), page=rng.choice([1, 2, 2, 16, 64]),
                  tokens=between(1, 40001))
    elif op == "norm":
        c = _norm("", dtype, kind=rng.choice(["rms", "rms", "layer"]), tokens=between(1, 8191), width=between(64, 16384),
                  block=rng.random() < 0.8)
        if rng.random() < 0.7:
            c["width"] = max(64, c["width"] // 64 * 64)
        if c["kind"] == "layer":
            c["bias"] = rng.random() < 0.7
        if c["block"]:
            c["post"] = rng.random() < 0.5
            c["gate"] = rng.choice(["none", "none", "channel", "token", "element"])
            c["residual_scale"] = rng.choice([1.0, 1.0, 1.5])
            c["block_scale"] = rng.choice([1.0, 1.0, 0.22])
    else:
        c = _attend("", dtype, q_heads=heads[0], kv_heads=heads[1], head_dim=rng.choice([32, 64, 96, 128, 128, 256]),
                    page=rng.choice([1, 2, 2, 16, 64]), weights=rng.random() < 0.2, lengths=rng.randrange(1 << 30))
        if rng.random() < 0.2:
            c["window"] = between(64, 4096)
        if rng.random() < 0.5:
            c["chunks"] = between(1, 16)
            c["chunk_max"] = between(2, 2048)
            c["chunk_min"] = between(2, c["chunk_max"])
            if rng.random() < 0.5:
                c["past_max"] = between(16, 32000)
                c["past_min"] = between(1, c["past_max"])
        if not c["chunks"] or rng.random() < 0.4:
            c["decode"] = between(1, 256)
            c["ctx_max"] = between(16, 64000)
            c["ctx_min"] = between(1, c["ctx_max"])
    while work(c)["bytes"] > MAX_BYTES or work(c)["flops"] > MAX_FLOPS:
        for k in ("decode", "chunks", "ctx_max", "past_max", "tokens"):
            if c.get(k, 0) > 1:
                c[k] = max(1, c[k] * 3 // 4)
        if op == "attend":
            c["ctx_min"], c["past_min"] = min(c["ctx_min"], c["ctx_max"]), min(c["past_min"], c["past_max"])
    del c["name"]
    return c


# ---- lengths: the case's own, the same for every seed of the inputs ----------------------------------------------------
def _spread(rng, lo, hi):
    return lo if hi <= lo else min(hi, int(round(max(lo, 1) * (hi / max(lo, 1)) ** rng.random())))


def _lengths(c):
    """(new tokens, cached tokens with the new ones) of each request."""
    rng = random.Random(c["lengths"])
    reqs = [(1, _spread(rng, c["ctx_min"], c["ctx_max"])) for _ in range(c["decode"])]
    for _ in range(c["chunks"]):
        n = _spread(rng, c["chunk_min"], c["chunk_max"])
        reqs.append((n, n + _spread(rng, c["past_min"], c["past_max"])))
    return reqs


def _visible(n, length, window):
    """(pairs of a new token and a cached token it sees, cached tokens that any of them sees)"""
    if window and window < length:
        return sum(min(p + 1, window) for p in range(length - n, length)), min(length, window + n - 1)
    return n * length - n * (n - 1) // 2, length


def work(case):
    c = case
    if c["op"] == "keep":
        w, hq, hk = c["tokens"] * c["head_dim"], c["q_heads"], c["kv_heads"]
        # q in and out, k and v in and back in 16 bits, their codes; their powers, a position and a slot a token
        return {"bytes": 2 * w * (2 * hq + 4 * hk) + 2 * w * hk + c["tokens"] * (2 * hk + 16), "flops": 3 * c["tokens"] * c["rotary_dim"] * (hq + hk)}
    if c["op"] == "read":
        w = c["tokens"] * c["head_dim"] * c["kv_heads"]
        return {"bytes": 2 * w + 4 * w + c["tokens"] * (2 * c["kv_heads"] + 8), "flops": 2 * w}
    if c["op"] == "norm":
        w = c["tokens"] * c["width"]
        each = 4 if c["block"] else 2                                         # x, block in; stream and normalised stream out
        gate = {"none": 0, "channel": c["width"], "token": c["tokens"], "element": w}[c["gate"]]
        vectors = (1 + c["bias"]) * (1 + c["post"]) * c["width"]
        return {"bytes": 2 * (each * w + gate + vectors), "flops": w * (4 + 4 * c["post"] + 2 * c["block"])}
    d, bytes_, flops = c["head_dim"], 0, 0
    for n, length in _lengths(c):
        pairs, seen = _visible(n, length, c["window"])
        bytes_ += 2 * 2 * n * c["q_heads"] * d + seen * c["kv_heads"] * (2 * d + 2) + 4 * -(-seen // c["page"])
        bytes_ += 8 * seen if c["weights"] else 0
        flops += 4 * d * c["q_heads"] * pairs
    return {"bytes": bytes_, "flops": flops}


# ---- inputs ------------------------------------------------------------------------------------------------------------
class _State:
    pass


def prepare(case, seed):
    c, s = case, _State()
    s.case = c
    s.g = torch.Generator(device=DEVICE).manual_seed(seed)
    s.rng = np.random.RandomState(seed % (1 << 31))
    {"keep": _prepare_keep, "read": _prepare_read, "attend": _prepare_attend, "norm": _prepare_norm}[c["op"]](c, s)
    return s


def _normal(s, dtype, *shape, std=1.0):
    return torch.empty(*shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=s.g)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _coded(s, c, pages):
    """A cache of 8-bit codes as earlier passes have left it: k with a few strong channels, as models have them."""
    hk, d, page = c["kv_heads"], c["head_dim"], c["page"]
    parts = []
    for std in (1.0 + 5.0 * (torch.rand(hk, 1, d, device=DEVICE, generator=s.g) > 0.96), 1.0):
        codes = torch.empty(pages, hk, page, d, dtype=torch.float8_e4m3fn, device=DEVICE)
        powers = torch.empty(pages, hk, page, dtype=torch.uint8, device=DEVICE)
        step = max(1, (1 << 27) // (hk * page * d))
        for at in range(0, pages, step):                                      # some hundred MB of 32-bit values at a time
            n = min(step, pages - at)
            code, e = _code(_normal(s, torch.float32, n, hk, page, d) * std, *POWERS[c["dtype"]])
            codes[at:at + n], powers[at:at + n] = code.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)
        parts.append((codes, powers))
    s.key_codes, s.value_codes = parts[0][0], parts[1][0]
    s.powers = torch.stack([parts[0][1], parts[1][1]], dim=-1).view(torch.float8_e8m0fnu)


def _prepare_keep(c, s):
    dtype, T, hq, hk, d = DTYPES[c["dtype"]], c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    qkv = _normal(s, dtype, T, (hq + 2 * hk) * d)                             # one projection's output, cut in three
    s.q, s.k, s.v = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hk * d, hk * d], dim=1))
    s.positions = torch.from_numpy(s.rng.randint(0, c["farthest"], T)).to(DEVICE)
    pages = -(-(T + max(16, T // 4)) // c["page"])
    _coded(s, c, pages)
    s.loc = torch.from_numpy(s.rng.permutation(pages * c["page"])[:T].astype(np.int64)).to(DEVICE)
    s.q_out = torch.empty(T, hq, d, dtype=dtype, device=DEVICE)
    if own:
        from valora_amd.rotary import Rotary
        s.rotary = Rotary(d, rotary_dim=c["rotary_dim"], interleaved=c["interleaved"], device=DEVICE)


def _prepare_read(c, s):
    pages = -(-c["tokens"] // c["page"]) + 16
    _coded(s, c, pages)
    order = torch.from_numpy(s.rng.permutation(pages)[:-(-c["tokens"] // c["page"])].astype(np.int64)).to(DEVICE)
    s.loc = (order[:, None] * c["page"] + torch.arange(c["page"], device=DEVICE)).flatten()[:c["tokens"]].contiguous()


def _prepare_attend(c, s):
    dtype, hq, hk, d, page = DTYPES[c["dtype"]], c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    s.reqs = _lengths(c)
    s.new, s.len = [n for n, _ in s.reqs], [l for _, l in s.reqs]
    T = sum(s.new)
    s.starts = [int(v) for v in np.cumsum(s.new) - np.array(s.new)]
    # pages of each request, scattered over the pool as they are after a while of serving
    counts = [-(-n // page) for n in s.len]
    pages = sum(counts) + max(4, sum(counts) // 16)
    order, table, at = s.rng.permutation(pages).astype(np.int32), np.full((len(counts), max(counts)), -1, dtype=np.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    s.table = torch.from_numpy(table).to(DEVICE)
    # heads differ in how sharply they look
    sharp = torch.linspace(0.3, 1.5, hq, device=DEVICE)[None, :, None]
    s.q = (_normal(s, torch.float32, T, hq, d) * sharp).to(dtype)
    _coded(s, c, pages)
    s.b_start_loc, s.b_seq_len, s.b_kv_len = _int32(s.starts), _int32(s.new), _int32(s.len)
    s.out = torch.empty(T, hq, d, dtype=dtype, device=DEVICE)
    s.weights = None
    if c["weights"]:
        s.weights = torch.rand(len(s.reqs), s.table.shape[1] * page, device=DEVICE, generator=s.g)
    if own:
        from valora_amd.attention import AttentionPlan
        s.plan = AttentionPlan(s.b_start_loc, s.b_seq_len, s.b_kv_len, n_tokens=T, max_seq_len=max(s.new), max_kv_len=max(s.len),
                               q_heads=hq, kv_heads=hk, head_dim=d, page_size=page, window=c["window"])


def _prepare_norm(c, s):
    dtype, T, H = DTYPES[c["dtype"]], c["tokens"], c["width"]
    channels = 1.0 + 20.0 * (torch.rand(H, device=DEVICE, generator=s.g) > 0.995)        # a residual stream has a few strong channels
    s.x = (_normal(s, torch.float32, T, H) * channels).to(dtype)
    s.weight = (1.0 + _normal(s, torch.float32, H, std=0.2)).to(dtype)
    s.bias = _normal(s, dtype, H, std=0.1) if c["bias"] else None
    s.block = _normal(s, dtype, T, H, std=0.7) if c["block"] else None
    s.block_weight = (1.0 + _normal(s, torch.float32, H, std=0.2)).to(dtype) if c["post"] else None
    s.block_bias = _normal(s, dtype, H, std=0.1) if c["post"] and c["bias"] else None
    shape = {"none": None, "channel": (H,), "token": (T, 1), "element": (T, H)}[c["gate"]]
    s.gate = None if shape is None else _normal(s, dtype, *shape, std=0.5)
    s.residual_out = torch.empty_like(s.x) if c["block"] else None
    s.out = torch.empty_like(s.x)


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state.case
    if not own:
        return {"keep": _plain_keep, "read": _plain_read, "attend": _plain_attend, "norm": _plain_norm}[c["op"]](s, c)
    if c["op"] == "keep":
        from valora_amd import cache8
        s.rotary.store8(s.positions, s.q, s.k, s.v, s.key_codes, s.value_codes, s.powers, s.loc, q_out=s.q_out)
        k, v = cache8.read(s.key_codes, s.value_codes, s.powers, s.loc, dtype=DTYPES[c["dtype"]])
        return s.q_out, k, v
    if c["op"] == "read":
        from valora_amd import cache8
        return cache8.read(s.key_codes, s.value_codes, s.powers, s.loc, dtype=DTYPES[c["dtype"]])
    if c["op"] == "norm":
        from valora_amd.norm import block_norm
        r, h = block_norm(s.x, s.weight, s.bias, block=s.block, block_weight=s.block_weight, block_bias=s.block_bias, gate=s.gate,
                          residual_scale=c["residual_scale"], block_scale=c["block_scale"], kind=c["kind"], eps=1e-5,
                          residual_out=s.residual_out, out=s.out)
        return (r, h) if c["block"] else h
    if s.weights is None:
        s.plan.attend8(s.out, s.q, s.key_codes, s.value_codes, s.powers, s.table)
        return s.out
    weights = s.weights.clone()
    s.plan.attend8(s.out, s.q, s.key_codes, s.value_codes, s.powers, s.table, weights=weights)
    return s.out, weights


# the plain form: elementary torch operations in 32 bits
def _power(e, dtype):
    """2^e to the last bit, from its bits"""
    if dtype == torch.float64:
        return ((e.long() + 1023) << 52).view(torch.float64)
    return ((e.int() + 127) << 23).view(torch.float32)


def _code(x, lowest, highest):
    """(the nearest e4m3 values of x / 2^e, e): e the least with which the largest of a head's elements is at most 448."""
    part, e = torch.frexp(x.abs().amax(-1))                                   # 448 = 0.875 * 2^9
    e = torch.where(part > 0, e - 9 + (part > 0.875).int(), lowest).clamp(lowest, highest)
    y = (x * _power(-e, x.dtype)[..., None]).clamp(-448.0, 448.0)
    step = _power(torch.frexp(y)[1].clamp(min=-5) - 4, x.dtype)               # three bits behind the first, 2^-9 below 2^-6
    return torch.round(y / step) * step, e


def _plain_values(codes, powers, slots):
    """What the codes of these slots [...] stand for, [..., kv heads, head_dim] in 32 bits."""
    page = codes.shape[2]
    at, off = slots // page, slots % page
    return codes.view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn).float() * powers.view(torch.uint8)[at, :, off].view(torch.float8_e8m0fnu).float()[..., None]


def _plain_rotate(x, cos, sin, R, interleaved):
    x = x.to(cos.dtype)
    out = x.clone()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        out[..., 0:R:2], out[..., 1:R:2] = ra, rb
    else:
        out[..., :R // 2], out[..., R // 2:R] = ra, rb
    return out


def _plain_keep(s, c):
    dtype, R, page = s.q.dtype, c["rotary_dim"], c["page"]
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEVICE) / R)
    angle = s.positions.double()[:, None] * inv[None]                         # far positions: 64 bits
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    s.q_out.copy_(_plain_rotate(s.q, cos.float(), sin.float(), R, c["interleaved"]).to(dtype))
    at, off = s.loc // page, s.loc % page
    back = []
    # (which of two codes is nearest is found in 64 bits)
    for x, codes, powers in ((_plain_rotate(s.k, cos, sin, R, c["interleaved"]), s.key_codes, s.powers[..., 0]), (s.v.float(), s.value_codes, s.powers[..., 1])):
        code, e = _code(x, *POWERS[c["dtype"]])
        codes.view(torch.uint8)[at, :, off] = code.to(torch.float8_e4m3fn).view(torch.uint8)
        powers.view(torch.uint8)[at, :, off] = (e + 127).to(torch.uint8)
        back.append(_plain_values(codes, powers, s.loc).to(dtype))
    return s.q_out, back[0], back[1]


def _plain_read(s, c):
    dtype = DTYPES[c["dtype"]]
    return _plain_values(s.key_codes, s.powers[..., 0], s.loc).to(dtype), _plain_values(s.value_codes, s.powers[..., 1], s.loc).to(dtype)


def _plain_norm(s, c):
    def norm(x, w, b):
        if c["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.float()
        return y if b is None else y + b.float()

    if not c["block"]:
        s.out.copy_(norm(s.x.float(), s.weight, s.bias))
        return s.out
    o = s.block.float()
    if c["post"]:
        o = norm(o, s.block_weight, s.block_bias)
    if s.gate is not None:
        o = o * s.gate.float()
    r = c["residual_scale"] * s.x.float() + c["block_scale"] * o
    s.residual_out.copy_(r)
    s.out.copy_(norm(r, s.weight, s.bias))
    return s.residual_out, s.out


def _plain_attend(s, c):
    weights = None if s.weights is None else s.weights.clone()
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    group = hq // hk
    # requests with as many new tokens side by side, as many as some hundred MB hold, padded to the longest
    order = sorted(range(len(s.reqs)), key=lambda b: s.reqs[b])
    at = 0
    while at < len(order):
        n, end = s.new[order[at]], at + 1
        while end < len(order) and s.new[order[end]] == n and (end + 1 - at) * s.len[order[end]] * hk * (group * n + 2 * d) <= 1 << 28:
            end += 1
        some = order[at:end]
        at, B, L = end, len(some), max(s.len[b] for b in some)
        which, length = torch.tensor(some, device=DEVICE), torch.tensor([s.len[b] for b in some], device=DEVICE)
        j = torch.arange(L, device=DEVICE)
        slots = s.table[which].long()[:, :-(-L // page)].clamp(min=0).repeat_interleave(page, 1)[:, :L] * page + j % page
        rows = torch.tensor([s.starts[b] for b in some], device=DEVICE)[:, None] + torch.arange(n, device=DEVICE)
        p = (length[:, None] - n + torch.arange(n, device=DEVICE))[..., None]
        seen = (j <= p) & ((j > p - c["window"]) if c["window"] else True)                       # [B, n, L]
        seen = seen[:, None, None].expand(B, 1, group, n, L).reshape(B, 1, group * n, L)
        K = _plain_values(s.key_codes, s.powers[..., 0], slots).transpose(1, 2)                  # [B, kv heads, L, d]
        V = _plain_values(s.value_codes, s.powers[..., 1], slots).transpose(1, 2)
        q = s.q[rows].float().view(B, n, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B, hk, group * n, d)
        step = max(1, (1 << 28) // (B * group * n * L))                                          # heads at a time
        for h in range(0, hk, step):
            score = torch.matmul(q[:, h:h + step] * d ** -0.5, K[:, h:h + step].transpose(2, 3).contiguous())
            score = score.masked_fill(~seen, -math.inf)
            e = torch.exp(score - score.amax(-1, keepdim=True))
            prob = e / e.sum(-1, keepdim=True)
            o = torch.matmul(prob, V[:, h:h + step].contiguous())                                # [B, heads, group * n, d]
            o = o.unflatten(2, (group, n)).permute(0, 3, 1, 2, 4).reshape(B, n, -1, d)
            s.out[rows, h * group:h * group + o.shape[2]] = o.to(s.out.dtype)
            if weights is not None:
                weights[which, :L] += prob.sum(dim=(1, 2))
    return s.out if weights is None else (s.out, weights)


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"keep": _exact_keep, "read": _exact_read, "attend": _exact_attend, "norm": _exact_norm}[case["op"]](s, case)


def _exact_codes(x, c):
    """Values of the 8-bit cache for heads x [..., d] in 64 bits: each goes to the nearest of all e4m3 values, to the even one of two."""
    lowest, highest = POWERS[c["dtype"]]
    powers = torch.tensor([2.0 ** e for e in range(lowest, highest + 1)], dtype=torch.float64, device=x.device)
    which = torch.searchsorted(448.0 * powers, x.abs().amax(-1, keepdim=True)).clamp(max=len(powers) - 1)
    power = powers[which]
    grid = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (k - 9) for k in range(15) for m in range(8)],
                        dtype=torch.float64, device=x.device)[:127]                              # 0 .. 448, the even ones at even places
    y = (x.abs() / power).clamp(max=448.0)
    hi = torch.searchsorted(grid, y).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y, y - grid[lo]
    near = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.sign(x) * grid[near] * power


def _exact_keep(s, c):
    R = c["rotary_dim"]
    freq = torch.tensor([10000.0 ** (-2.0 * i / R) for i in range(R // 2)], dtype=torch.float64)
    turn = torch.outer(s.positions.cpu().double(), freq).to(DEVICE)
    z = torch.polar(torch.ones_like(turn), turn)[:, None]                     # a pair as a complex number

    def rotate(x):
        x = x.double()
        head = x[..., :R]
        pairs = head.unflatten(-1, (R // 2, 2)) if c["interleaved"] else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat([y, x[..., R:]], dim=-1)

    return rotate(s.q), _exact_codes(rotate(s.k), c), _exact_codes(s.v.double(), c)


def _exact_values(codes, powers, slots):
    """[slots, kv heads, d]: each code's bits taken apart"""
    at, off = torch.div(slots, codes.shape[2], rounding_mode="floor"), torch.remainder(slots, codes.shape[2])
    rows = codes.view(torch.uint8)[at, :, off].long()
    two = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64, device=codes.device)
    field, m = (rows >> 3) & 15, (rows & 7).double()
    size = torch.where(field == 0, m * 2.0 ** -9, (8.0 + m) * two[field + 117])
    return torch.where(rows >= 128, -size, size) * two[powers.view(torch.uint8)[at, :, off].long()][..., None]


def _exact_read(s, c):
    return _exact_values(s.key_codes, s.powers[..., 0], s.loc), _exact_values(s.value_codes, s.powers[..., 1], s.loc)


def _exact_norm(s, c):
    def norm(x, w, b):
        if c["kind"] == "layer":
            var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
            y = (x - mean) / torch.sqrt(var + 1e-5) * w.double()
        else:
            y = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + 1e-5) * w.double()
        return y if b is None else y + b.double()

    if not c["block"]:
        return norm(s.x.double(), s.weight, s.bias)
    o = s.block.double()
    o = norm(o, s.block_weight, s.block_bias) if c["post"] else o
    g = 1.0 if s.gate is None else s.gate.double()
    r = s.x.double() * c["residual_scale"] + o * g * c["block_scale"]
    return r, norm(r, s.weight, s.bias)


def _exact_attend(s, c):
    if work(c)["flops"] > 2e12:
        return None
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    weights = None if s.weights is None else s.weights.double()
    for b, (n, length) in enumerate(s.reqs):
        slots = (s.table[b].long()[:, None] * page + torch.arange(page, device=DEVICE)).reshape(-1)[:length]
        last = torch.arange(length - n, length, device=DEVICE)
        j = torch.arange(length, device=DEVICE)
        hidden = (j[None] > last[:, None]) | (j[None] <= last[:, None] - (c["window"] or length + 1))
        K, V = _exact_values(s.key_codes, s.powers[..., 0], slots), _exact_values(s.value_codes, s.powers[..., 1], slots)
        if n == 1:                                                             # all heads of a lone token at once
            q = s.q[s.starts[b]].double().view(hk, hq // hk, d)
            score = (torch.matmul(K.transpose(0, 1).contiguous(), q.transpose(1, 2).contiguous()) / math.sqrt(d)).masked_fill(hidden.view(1, length, 1), -math.inf)
            prob = torch.softmax(score, dim=1)                                 # [kv heads, length, heads of a group]
            out[s.starts[b]] = torch.matmul(prob.transpose(1, 2).contiguous(), V.transpose(0, 1).contiguous()).reshape(hq, d)
            if weights is not None:
                weights[b, :length] += prob.sum(dim=(0, 2))
            continue
        for h in range(hq):
            q = s.q[s.starts[b]:s.starts[b] + n, h].double()
            kv = h * hk // hq
            score = (q @ K[:, kv].T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf)
            prob = torch.softmax(score, dim=-1)
            out[s.starts[b]:s.starts[b] + n, h] = prob @ V[:, kv].contiguous()
            if weights is not None:
                weights[b, :length] += prob.sum(0)
    return out if weights is None else (out, weights)
