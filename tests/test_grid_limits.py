"""Calls whose launch would have more than 2^32 threads along a dimension, which a launch leaves out without an error, are refused where they are not cut
in parts.  Through the C ABI with addresses that nothing is read from."""
from tests.test_attention_refusals import plan
from tests.test_cache8_refusals import A, cache
from valora_amd import _lib


def test_attention():
    L = _lib.lib()
    p = plan(n_req=1 << 20, n_tokens=1 << 20, max_seq_len=1, max_kv_len=16, q_heads=16, kv_heads=16, head_dim=32)
    p.dev, p.bytes = A, L.mlora_attention_plan_bytes(p)
    for call in (lambda: L.mlora_paged_attention(None, p, A, 1 << 40, A, 512, A, 512, A, 512, A, 512, 1 << 20, A, 1, 1, 1.0, None, 0, 0),
                 lambda: L.mlora_paged_attention_codes(None, p, A, 1 << 40, A, 512, A, 512,
                                                       cache(kv_heads=16, head_dim=32, key_stride=8192, value_stride=8192, powers_stride=512), A, 1, 1,
                                                       1.0, None, 0, 0)):
        assert call() == -2 and b"too many tiles" in L.mlora_last_error(), L.mlora_last_error()


def test_eviction():
    L = _lib.lib()
    assert L.mlora_cache_evict(None, A, 4, A, A, 4, 1 << 22, 4, 1, 3, 1, 0, A, A, A, A) == -2 and b"requests" in L.mlora_last_error()


def test_pool_rows():
    L = _lib.lib()
    for call in (L.mlora_pool_gather_rows, L.mlora_pool_scatter_rows):
        assert call(None, A, 1 << 30, 0, A, 0, A, 4 << 24, 16, 1) == -1 and b"too many rows" in L.mlora_last_error()
