"""What the attention block's entry points refuse before anything is launched: the C ABI's checks and those of the Python side,
without a GPU."""
import ctypes
import math

import pytest
import torch

from valora_amd import _lib
from valora_amd.rotary import frequencies


def plan(**kw):
    p = dict(dev=None, bytes=0, n_req=3, n_tokens=8, max_seq_len=4, max_kv_len=1000, q_heads=8, kv_heads=2, head_dim=128, page_size=16, window=0)
    p.update(kw)
    return _lib.AttentionPlan(*[p[n] for n, _ in _lib.AttentionPlan._fields_])


def test_plan_shapes():
    L = _lib.lib()
    assert L.mlora_attention_plan_bytes(plan()) > 0 and L.mlora_attention_workspace_bytes(plan(), 0) > 0
    # a cache that no request can fill beyond one piece needs no room for pieces, with weights a logarithm a row
    assert L.mlora_attention_workspace_bytes(plan(max_kv_len=128), 0) == 0
    assert L.mlora_attention_workspace_bytes(plan(max_kv_len=128), 1) == 8 * 8 * 4 + 3 * 16 * 2 * 128 * 4      # and scores
    assert L.mlora_attention_workspace_bytes(plan(n_req=4096, n_tokens=4096, max_kv_len=100000), 1) <= (256 << 20) + (64 << 20)
    for kw, message in ((dict(q_heads=7), b"multiple of kv_heads"), (dict(kv_heads=0), b"kv_heads=0"), (dict(head_dim=100), b"head_dim=100"),
                        (dict(head_dim=512), b"head_dim=512"), (dict(page_size=12), b"page_size=12"), (dict(page_size=512), b"page_size=512"),
                        (dict(page_size=0), b"page_size=0"), (dict(n_req=-1), b"negative"), (dict(window=-1), b"negative"),
                        (dict(max_kv_len=1 << 31), b"too large"),
                        (dict(n_tokens=1 << 40), b"too large"), (dict(n_tokens=1 << 62), b"too large"),
                        (dict(n_req=1 << 20, max_kv_len=1 << 30), b"too large")):
        assert L.mlora_attention_plan_bytes(plan(**kw)) == 0 and message in L.mlora_last_error(), kw
        assert L.mlora_attention_workspace_bytes(plan(**kw), 1) == 0
        assert L.mlora_build_attention_plan(None, plan(**kw), None, None, None) < 0


def cut_few(spans, hkv):
    """Records, slots and joins of the few-rows list, as the plan kernel cuts it."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    piece = max(128, up(up(sum(spans) * hkv, 1024), 64) * 64)
    ks = [1 if s <= piece else up(s, up(up(s, up(s, piece)), 64) * 64) for s in spans]
    return sum(ks), sum(k for k in ks if k > 1), sum(k > 1 for k in ks)


def cut_tall(spans, shares):
    """(records, slots, joins, pieces per tile, first record of each share) of the tall list, as the plan kernel cuts it."""
    least, overhead = 512, 192
    if shares is None:        # none can be cut: a share a tile
        return len(spans), 0, 0, [[s] for s in spans], list(range(len(spans)))
    line = sum(s + overhead for s in spans)
    n = min(-(-line // least), shares)
    share = -(-line // n) if n else 1
    n = -(-line // share)
    at, pieces, first, records = 0, [], {}, 0
    for s in spans:
        ends, last, j = [], 0, -(-at // share)
        marks = []
        while j * share < at + s + overhead:
            inside = j * share - at - overhead // 2
            cut = int((inside + 32) / 64) * 64
            if inside < least // 2 or s < least:
                cut = 0 if inside * 2 < s else s
            elif inside > s - least // 2:
                cut = s
            if last < cut < s:
                ends.append(cut)
                last = cut
            marks.append((j, None if cut >= s and s > 0 else len(ends)))
            j += 1
        k = len(ends) + 1
        for j, i in marks:
            first[j] = records + (k if i is None else i)
        pieces.append([b - a for a, b in zip([0] + ends, ends + [s])])
        records += k
        at += s + overhead
    return records, sum(len(p) for p in pieces if len(p) > 1), sum(len(p) > 1 for p in pieces), pieces, [first[j] for j in range(n)]


def test_the_lists_hold_any_batch_the_bounds_allow():
    """The records that the plan kernel would write, counted as it counts them, against the room the plan has: requests of all kinds
    and lengths within n_tokens, max_seq_len and max_kv_len; and the shares, which are even up to what is not cut."""
    import random
    L, rng = _lib.lib(), random.Random(1)
    for _ in range(400):
        hkv, group = rng.choice([1, 2, 8, 32, 40]), rng.choice([1, 4, 7, 8])
        n_req, max_seq, max_kv = rng.randint(1, 300), rng.choice([1, 2, 5, 40, 900]), rng.choice([1, 64, 256, 300, 511, 512, 5000, 70000])
        new = [rng.choice([0, 1, 1, rng.randint(1, max_seq)]) for _ in range(n_req)]
        kv = [rng.randint(0, max_kv) if rng.random() < 0.8 else max_kv for _ in range(n_req)]
        few, tall = [], []
        for n, l in zip(new, kv):
            rows = n * group
            if 0 < rows <= 16:
                few.append(max(0, l))
            else:
                tall += [max(0, l - n + (min(r + 128, rows) - 1) // group + 1) for r in range(0, rows, 128)]
        p = plan(n_req=n_req, n_tokens=max(1, sum(new)), max_seq_len=max_seq, max_kv_len=max_kv, q_heads=hkv * group, kv_heads=hkv)
        words, room = L.mlora_attention_plan_bytes(p) // 4, L.mlora_attention_workspace_bytes(p, 0)
        shares = 512 // hkv if max_kv >= 512 else None
        f, t = cut_few(few, hkv), cut_tall(tall, shares)
        need = 32 + 8 * (f[0] + t[0] + f[2] + t[2] + n_req) + len(t[4]) + 1 + hkv * f[2]
        assert need <= words, (f, t[:3], words)
        assert (f[1] * 16 + t[1] * 128) * hkv * (128 + 4) * 4 <= room, (f, t[:3], room)
        assert all(sum(p) == s and (len(p) == 1 or min(p) >= 192) for p, s in zip(t[3], tall))
        if t[4] and shares is not None:
            assert t[4][0] == 0 and t[4] == sorted(t[4]) and t[4][-1] <= t[0]
            flat = [x + (192 if i == 0 else 0) for q in t[3] for i, x in enumerate(q)]
            share = -(-sum(flat) // len(t[4]))
            bounds = t[4] + [t[0]]
            # a share is off by what its two ends are moved: half of what is not cut, and the start of a tile
            assert all(sum(flat[a:b]) <= share + 512 + 192 + 128 for a, b in zip(bounds, bounds[1:]))


def test_attention_arguments():
    L = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    at = (ctypes.addressof(buf) + 255) & ~255
    p = plan(dev=at, bytes=1 << 15)
    ok = dict(ws=at, ws_bytes=1 << 40, out=at, out_stride=1024, q=at + 256, q_stride=1024, k=at, k_stride=256, v=at, v_stride=256, rows=64, table=at,
              table_stride=63, table_width=63, scale=0.1, weights=None, w_stride=0, dtype=0)

    def call(plan=p, **kw):
        a = dict(ok, **kw)
        return L.mlora_paged_attention(None, plan, a["ws"], a["ws_bytes"], a["out"], a["out_stride"], a["q"], a["q_stride"], a["k"], a["k_stride"],
                                       a["v"], a["v_stride"], a["rows"], a["table"], a["table_stride"], a["table_width"], a["scale"], a["weights"],
                                       a["w_stride"], a["dtype"])

    for kw, code, message in ((dict(dtype=2), -2, b"dtype=2"), (dict(scale=0.0), -1, b"scale"), (dict(scale=-1.0), -1, b"scale"), (dict(scale=math.nan), -1, b"scale"),
                              (dict(q_stride=1000), -1, b"shorter"), (dict(q_stride=1028), -1, b"16 bytes"), (dict(k=at + 8), -1, b"16-byte"),
                              (dict(v_stride=128), -1, b"shorter"), (dict(table_width=62, table_stride=62), -1, b"needs 63"), (dict(table_stride=62), -1, b"table"),
                              (dict(rows=15), -1, b"no page"), (dict(rows=-1), -2, b"pool rows"), (dict(k=None), -1, b"no page"), (dict(q=None), -1, b"null"),
                              (dict(table=None), -1, b"null"), (dict(ws_bytes=100), -3, b"workspace"), (dict(ws=None), -3, b"workspace"),
                              (dict(ws=at + 16), -3, b"workspace"), (dict(weights=at, w_stride=999), -1, b"weights"), (dict(k_stride=1 << 31), -2, b"2 GB")):
        assert call(**kw) == code and message in L.mlora_last_error(), (kw, L.mlora_last_error())
    assert call(plan=plan(dev=at, bytes=64)) == -3 and call(plan=plan(dev=None, bytes=1 << 15)) == -3
    assert call(plan=plan(dev=at, bytes=1 << 15, n_req=0)) == 0 and call(plan=plan(dev=at, bytes=1 << 15, n_tokens=0)) == 0
    assert L.mlora_build_attention_plan(None, plan(dev=at, bytes=64), at, at, at) == -3
    assert L.mlora_build_attention_plan(None, p, None, at, at) == -1


def test_rotary_and_evict_arguments():
    L = _lib.lib()
    part = lambda **kw: _lib.RotaryPart(*[dict(dict(src=4096, dst=4096, src_token_stride=128, src_head_stride=64, dst_token_stride=128,  # noqa: E731
                                                    dst_head_stride=64, heads=2, flags=1), **kw)[n] for n, _ in _lib.RotaryPart._fields_])
    rot = lambda p, n=1, pos=64, loc=None, rows=0, T=3, d=64, r=64, f=64, dt=0: L.mlora_rotary(None, p, n, pos, loc, rows, T, d, r, 0, f, 1.0, dt)  # noqa: E731
    for kw, code, message in ((dict(n=0), -1, b"n_parts=0"), (dict(n=4), -1, b"n_parts=4"), (dict(T=-1), -1, b"T=-1"), (dict(dt=2), -2, b"dtype"), (dict(r=63), -2, b"rotary_dim=63"),
                              (dict(r=66), -2, b"rotary_dim=66"), (dict(r=0), -2, b"rotary_dim=0"), (dict(pos=None), -1, b"null"), (dict(f=None), -1, b"null")):
        assert rot(part(), **kw) == code and message in L.mlora_last_error(), kw
    assert rot(part(flags=3)) == -1 and b"loc" in L.mlora_last_error()
    for kw in (dict(dst_token_stride=0), dict(dst_head_stride=0), dict(dst_head_stride=63)):
        assert rot(part(**kw)) == -1 and b"overlap" in L.mlora_last_error(), kw
    assert rot(part(flags=3, dst_token_stride=0), loc=64, rows=5) == -1 and b"overlap" in L.mlora_last_error()
    assert rot(part(src=None)) == -1 and rot(part(heads=-1)) == -1 and rot(part(heads=0)) == 0 and rot(part(), T=0) == 0
    ev = lambda n=2, width=10, page=1, budget=4, recent=1, sinks=0, ts=10, ws=None, t=64, out=64: L.mlora_cache_evict(  # noqa: E731
        None, t, ts, 64, 64, width * page if ws is None else ws, n, width, page, budget, recent, sinks, out, 64, 64, 64)
    for kw, code, message in ((dict(n=-1), -1, b"negative"), (dict(page=3), -2, b"page_size=3"), (dict(page=512), -2, b"page_size=512"), (dict(recent=0), -1, b"recent=0"),
                              (dict(budget=0), -1, b"budget=0"), (dict(sinks=-1), -1, b"sinks=-1"), (dict(sinks=4), -1, b"budget=4"), (dict(ts=9), -1, b"shorter"),
                              (dict(ws=9), -1, b"shorter"), (dict(t=None), -1, b"null"), (dict(out=None), -1, b"null"), (dict(width=1 << 30, page=256, ts=1 << 30), -2, b"2^31"),
                              (dict(width=1 << 55, page=256, ts=1 << 55, ws=1 << 55), -2, b"2^31")):
        assert ev(**kw) == code and message in L.mlora_last_error(), kw
    assert ev(n=0) == 0


def test_cpu_tensors_are_refused():
    from valora_amd.attention import AttentionPlan
    from valora_amd.kv_cache import evict
    from valora_amd.rotary import Rotary
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        AttentionPlan(i, i, i, 2, 1, 10, 4, 4, 64)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        evict(i.view(1, 2), i[:1], torch.zeros(1, 2), 1, 1)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        Rotary(64, device="cpu")


def test_rotary_frequencies():
    plain, gain = frequencies(8, 10000.0)
    assert plain == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15) and gain == 1.0
    assert frequencies(8, 10000.0, dict(type="linear", factor=4.0))[0] == pytest.approx([f / 4 for f in plain], rel=1e-15)
    ntk = frequencies(8, 10000.0, dict(type="ntk", factor=4.0))[0]
    assert ntk[0] == 1.0 and ntk[3] == pytest.approx(plain[3] / 4, rel=1e-14)       # the highest kept, the lowest divided
    bands = frequencies(8, 10000.0, dict(type="bands", factor=8.0, low=1.0, high=4.0, original_max_position=1000))[0]
    # 1000 tokens: 159 turns, 15.9, 1.59, 0.159
    assert bands[:2] == plain[:2] and bands[3] == plain[3] / 8
    t = (1000 * plain[2] / (2 * math.pi) - 1) / 3
    assert bands[2] == pytest.approx(plain[2] * t + plain[2] / 8 * (1 - t), rel=1e-14)
    yarn, gain = frequencies(128, 10000.0, dict(type="yarn", factor=4.0, original_max_position=4096))
    full = frequencies(128)[0]
    assert gain == pytest.approx(0.1 * math.log(4) + 1) and yarn[0] == full[0] and yarn[-1] == pytest.approx(full[-1] / 4)
    assert all(f / 4 * (1 - 1e-12) <= y <= f for f, y in zip(full, yarn)) and yarn == sorted(yarn, reverse=True)
    assert frequencies(128, scaling=dict(type="yarn", factor=4.0, original_max_position=4096, attention_factor=1.0))[1] == 1.0
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, scaling=dict(type="other", factor=2.0)),
               dict(rotary_dim=8, scaling=dict(type="linear")), dict(rotary_dim=8, scaling=dict(type="linear", factor=-1.0)), dict(rotary_dim=2, scaling=dict(type="ntk", factor=2.0)),
               dict(rotary_dim=8, scaling=dict(type="bands", factor=2.0)), dict(rotary_dim=8, scaling=dict(type="linear", factor=2.0, extra=1)),
               dict(rotary_dim=8, scaling=dict(type="bands", factor=2.0, low=4.0, high=1.0, original_max_position=10)),
               dict(rotary_dim=8, scaling=dict(type="bands", factor=2.0, original_max_position=0)), dict(rotary_dim=8, base=1.0, scaling=dict(type="yarn", factor=2.0, original_max_position=10)),
               dict(rotary_dim=8, scaling=dict(type="yarn", factor=2.0, original_max_position=10, beta_slow=0.0))):
        with pytest.raises(RuntimeError):
            frequencies(**kw)
