"""What the 8-bit cache's and the norms' entry points refuse before anything is launched, and the 8-bit cache's bookkeeping, without a GPU."""
import ctypes

import pytest
import torch

from tests.test_attention_refusals import plan
from tests.test_kv_cache_step import Plan, Pool, Turn, state
from valora_amd import _lib, cache8, kv_cache
from valora_amd.kv_cache import KVCache
from valora_amd.layer import LayerWeights, layer_forward
from valora_amd.norm import block_norm

A = 1 << 20      # an address that nothing is read from


def cache(**kw):
    c = dict(key_codes=A, value_codes=A + (1 << 24), powers=A + (1 << 25), n_pages=10, key_stride=2 * 16 * 128, value_stride=2 * 16 * 128,
             powers_stride=2 * 16 * 2, kv_heads=2, head_dim=128, page_size=16)
    c.update(kw)
    return _lib.Cache8(*[c[n] for n, _ in _lib.Cache8._fields_])


CACHES = [(dict(head_dim=80), -2, b"head_dim=80"), (dict(head_dim=512), -2, b"head_dim=512"), (dict(page_size=12), -2, b"page_size=12"),
          (dict(page_size=0), -2, b"page_size=0"), (dict(page_size=512), -2, b"page_size=512"), (dict(kv_heads=0), -1, b"kv_heads=0"),
          (dict(kv_heads=1025), -1, b"kv_heads=1025"), (dict(n_pages=-1), -2, b"n_pages=-1"), (dict(n_pages=1 << 31), -2, b"out of range"),
          (dict(key_stride=4095), -1, b"shorter"), (dict(value_stride=4080), -1, b"shorter"), (dict(powers_stride=62), -1, b"shorter"),
          (dict(key_stride=1 << 31), -2, b"above 2 GB"), (dict(key_stride=4104), -1, b"16-byte"), (dict(value_codes=A + 8), -1, b"16-byte"),
          (dict(powers=A + 1), -1, b"2-byte"), (dict(powers_stride=65), -1, b"2-byte")]


def store(c, q=None, T=3, rotary_dim=128, dtype=0, k=A, loc=A, positions=A, freqs=A):
    return _lib.lib().mlora_rotary_store_codes(None, q, k, 256, 128, A, 256, 128, c, positions, loc, T, rotary_dim, 0, freqs, 1.0, dtype)


def read(c, n=3, k=A, v=A + 4096, k_stride=256, v_stride=256, dtype=0, loc=A):
    return _lib.lib().mlora_cache_read_codes(None, c, loc, n, k, k_stride, v, v_stride, dtype)


@pytest.mark.parametrize("kw,rc,message", CACHES)
def test_caches(kw, rc, message):
    L = _lib.lib()
    for call in (store, read):
        assert call(cache(**kw)) == rc and message in L.mlora_last_error(), kw


def test_attention_over_codes():
    L = _lib.lib()
    p = plan()
    p.dev, p.bytes = A, L.mlora_attention_plan_bytes(p)

    def call(c, p=p, q_stride=1024, table_width=63, scale=1.0, dtype=0, q=A, bytes_=1 << 40, weights=None, weights_stride=0):
        return L.mlora_paged_attention_codes(None, p, A, bytes_, A, 1024, q, q_stride, c, A, table_width, table_width, scale, weights, weights_stride, dtype)

    for kw, rc, message in CACHES:
        if not {"head_dim", "page_size", "kv_heads"} & set(kw):
            assert call(cache(**kw)) == rc and message in L.mlora_last_error(), kw
    for kw in (dict(head_dim=64), dict(page_size=8), dict(kv_heads=4)):
        assert call(cache(**kw)) == -1 and b"not 2 of 128 in pages of 16" in L.mlora_last_error()
    for kw, rc, message in ((dict(q_stride=1000), -1, b"shorter"), (dict(q_stride=1028), -1, b"16 bytes"), (dict(q=A + 2), -1, b"16 bytes"),
                            (dict(table_width=62), -1, b"max_kv_len=1000 needs 63"), (dict(scale=0.0), -1, b"positive"),
                            (dict(scale=float("nan")), -1, b"positive"), (dict(dtype=2), -2, b"dtype=2"), (dict(q=None), -1, b"null pointer"),
                            (dict(bytes_=64), -3, b"workspace has 64 bytes"), (dict(weights=A, weights_stride=999), -1, b"weights is shorter")):
        assert call(cache(), **kw) == rc and message in L.mlora_last_error(), kw
    for kw in (dict(n_pages=0), dict(key_codes=0), dict(powers=0)):
        assert call(cache(**kw)) == -1 and b"holds no page" in L.mlora_last_error()
    assert call(None) == -1 and b"cache is null" in L.mlora_last_error()
    none = plan(n_req=0, dev=A, bytes=1 << 20)
    assert call(cache(n_pages=0, key_codes=0, value_codes=0, powers=0), none) == 0


def test_store():
    L = _lib.lib()
    for kw, rc, message in ((dict(T=-1), -1, b"T=-1"), (dict(T=1 << 31), -2, b"2^31 - 1 tokens"), (dict(rotary_dim=3), -2, b"rotary_dim=3"),
                            (dict(rotary_dim=130), -2, b"rotary_dim=130"), (dict(rotary_dim=0), -2, b"rotary_dim=0"), (dict(dtype=7), -2, b"dtype=7"),
                            (dict(k=None), -1, b"null pointer"), (dict(loc=None), -1, b"null pointer"), (dict(positions=None), -1, b"null pointer"),
                            (dict(freqs=None), -1, b"null pointer")):
        assert store(cache(), **kw) == rc and message in L.mlora_last_error(), kw
    part = lambda **kw: _lib.RotaryPart(*[dict(dict(src=A, dst=A, src_token_stride=512, src_head_stride=128, dst_token_stride=512,  # noqa: E731
                                                    dst_head_stride=128, heads=4, flags=1), **kw)[n] for n, _ in _lib.RotaryPart._fields_])
    for kw, message in ((dict(dst_head_stride=64), b"overlap"), (dict(dst_token_stride=256), b"overlap"), (dict(heads=-1), b"heads=-1"),
                        (dict(src=None), b"null pointer")):
        assert store(cache(), part(**kw)) == -1 and message in L.mlora_last_error(), kw
    # keys' and values' codes: in each other's pages, and one before the other with room and without
    w = 2 * 16 * 128
    for kw in (dict(value_codes=A), dict(value_codes=A + 16), dict(value_codes=A + 9 * w), dict(value_codes=A + w, key_stride=3 * w, value_stride=2 * w),
               dict(value_codes=A + w - 16, key_stride=2 * w, value_stride=2 * w), dict(key_codes=A + w + 16, value_codes=A, key_stride=2 * w, value_stride=2 * w)):
        assert store(cache(**kw)) == -1 and b"keys and values overlap" in L.mlora_last_error(), kw
    assert store(cache(value_codes=A + 16), T=0) == -1
    assert store(cache(value_codes=A + w, key_stride=2 * w, value_stride=2 * w), T=0) == 0
    assert store(cache(value_codes=A + 10 * w), T=0) == 0
    assert store(cache(powers=0)) == -1 and b"null pointer" in L.mlora_last_error()


def test_read():
    L = _lib.lib()
    for kw, rc, message in ((dict(n=-1), -1, b"n=-1"), (dict(k_stride=255), -1, b"overlap"), (dict(v_stride=248), -1, b"overlap"),
                            (dict(k_stride=260), -1, b"16-byte"), (dict(v=A + 2), -1, b"16-byte"), (dict(dtype=5), -2, b"dtype=5"),
                            (dict(loc=None), -1, b"null pointer"), (dict(k=0), -1, b"null pointer"), (dict(n=1 << 60), -2, b"too large")):
        assert read(cache(), **kw) == rc and message in L.mlora_last_error(), kw
    assert read(cache(key_codes=0)) == -1 and b"null pointer" in L.mlora_last_error()
    assert read(cache(), n=0, loc=None) == 0


def norm(**kw):
    n = dict(x=A, block=A + (1 << 20), x_stride=64, block_stride=64, weight=A + (1 << 21), bias=None, block_weight=None, block_bias=None, gate=None,
             gate_row_stride=0, gate_column_stride=1, residual_out=A + (1 << 22), out=A + (1 << 23), residual_stride=64, out_stride=64, T=4, H=64,
             residual_scale=1.0, block_scale=1.0, eps=1e-6, offset=0.0, layer=0, f32=0)
    n.update(kw)
    return _lib.Norm(*[n[f] for f, _ in _lib.Norm._fields_])


def test_norm():
    L = _lib.lib()
    for kw, rc, message in ((dict(T=-1), -2, b"T=-1"), (dict(T=1 << 31), -2, b"out of range"), (dict(H=0), -2, b"H=0"), (dict(H=32769), -2, b"H=32769"),
                            (dict(eps=-1.0), -1, b"negative"), (dict(eps=float("nan")), -1, b"negative"), (dict(x=None), -1, b"null pointer"),
                            (dict(out=None), -1, b"null pointer"), (dict(block=None), -1, b"without block"),
                            (dict(block=None, residual_out=None, gate=A), -1, b"without block"),
                            (dict(block_bias=A), -1, b"without block_weight"), (dict(weight=None, bias=A), -1, b"bias without weight"),
                            (dict(weight=None, residual_out=None), -1, b"null pointer"), (dict(gate=A, gate_column_stride=2), -1, b"contiguous, or one"),
                            (dict(out_stride=63), -1, b"rows of a result"), (dict(residual_stride=63), -1, b"rows of a result"),
                            (dict(out=A + 128), -1, b"other rows"), (dict(out=A, out_stride=65), -1, b"other rows"), (dict(out=A - 2), -1, b"other rows"),
                            (dict(residual_out=A + (1 << 20) + 128), -1, b"other rows"), (dict(out=A + (1 << 22)), -1, b"results overlap"),
                            (dict(out=A + (1 << 22) + 64), -1, b"results overlap"),
                            (dict(gate=A + (1 << 23), gate_row_stride=64), -1, b"gate"), (dict(gate=A + (1 << 22) + 10), -1, b"gate"),
                            (dict(bias=A + (1 << 23)), -1, b"vector"), (dict(weight=A + (1 << 22) + 4 * 128 - 2), -1, b"vector")):
        assert L.mlora_block_norm(None, norm(**kw), 0) == rc and message in L.mlora_last_error(), (kw, L.mlora_last_error())
    assert L.mlora_block_norm(None, norm(), 3) == -2 and b"dtype=3" in L.mlora_last_error()
    assert L.mlora_block_norm(None, None, 0) == -1
    assert L.mlora_block_norm(None, norm(T=0), 0) == 0


def test_python_side():
    x = torch.zeros(2, 8, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="unknown norm"):
        block_norm(x, x[0], kind="batch")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        block_norm(x, x[0])
    codes = torch.zeros(2, 1, 2, 32, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        cache8.read(codes, codes, cache8.new_powers((2, 1, 2), "cpu"), torch.zeros(1, dtype=torch.long), torch.float16)
    z = torch.zeros(4, 4)
    w = LayerWeights(z, z, z, z, z, z, z, z[0], z[0], gate1=z[0])
    with pytest.raises(RuntimeError, match="fused=True"):
        layer_forward(z, w, None, None, lambda q, k, v: q, 1)
    with pytest.raises(RuntimeError, match="16-bit rows"):
        cache8.codes_of_rows(torch.zeros(3, 2, 64)[..., ::2].half()[..., ::2])


def make(monkeypatch, **kw):
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    return KVCache(Pool(), **dict(dict(max_requests=3, max_len=91, q_heads=4, rotary=Turn(), codes=True), **kw))


def test_two_tokens_a_row(monkeypatch):
    c = make(monkeypatch)
    assert c.table.shape == (3, 46) and c.powers.shape == (1, 100, 2, 2, 2)
    a = c.step([0, 2], [5, 2])                            # rows 0 1 2 | 3
    assert a.loc.tolist() == [0, 1, 2, 3, 4, 6, 7] and c.mem.can_use_mem_size == 96
    b = c.step([2, 0, 1], [3, 1, 1])                      # rows 4 5 | the second half of row 2 | row 6
    assert b.loc.tolist() == [8, 9, 10, 5, 12] and b.positions.tolist() == [2, 3, 4, 5, 0]
    assert c.lens == [6, 1, 5] and c.mem.can_use_mem_size == 93
    assert c.table[0, :4].tolist() == [0, 1, 2, -1] and c.table[2, :4].tolist() == [3, 4, 5, -1] and c.table[1, :2].tolist() == [6, -1]
    d = c.step([1, 2], [1, 1])                            # both have room: no row at all
    assert d.loc.tolist() == [13, 11] and c.mem.can_use_mem_size == 93
    with pytest.raises(RuntimeError, match="max_len=91"):
        c.step([0], [86])


def test_a_step_that_raises_changes_nothing(monkeypatch):
    c = make(monkeypatch)
    c.step([0, 1], [5, 3])
    before = state(c)
    with pytest.raises(Exception, match="pool space"):
        c.mem.can_use_mem_size, keep = 2, c.mem.can_use_mem_size
        try:
            c.step([0, 2], [2, 5])
        finally:
            c.mem.can_use_mem_size = keep
    assert state(c) == before
    cat = torch.cat
    with monkeypatch.context() as m:
        def broken(*a, **kw):
            raise torch.OutOfMemoryError("no memory")
        m.setattr(torch, "cat", broken)
        with pytest.raises(torch.OutOfMemoryError):
            c.step([0, 2], [2, 5])
    assert torch.cat is cat and state(c) == before
    assert c.step([0], [1]).loc.tolist() == [5]


def test_eviction_goes_by_rows(monkeypatch):
    c = make(monkeypatch, track=True)
    assert c.weights.shape == (3, 92)
    c.step([0, 1, 2], [11, 4, 12])
    calls = []
    monkeypatch.setattr(kv_cache, "evict", lambda t, l, w, *a: (calls.append((l.tolist(), a)), (t, l, w, t))[1])
    freed = []
    monkeypatch.setattr(KVCache, "_free", lambda self, rows, count: freed.append(count))
    assert c.evict(budget=9, recent=3, sinks=1) == 2 + 2
    assert calls == [([11, 4, 12], (4, 2, 1, 2))] and freed == [4] and c.lens == [7, 4, 8]
    # what the function refuses it is asked as it was given
    c.evict(budget=20, recent=0, sinks=-3)
    assert calls[-1][1] == (10, 0, -3, 2)
