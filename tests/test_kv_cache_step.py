"""The cache's bookkeeping without a GPU, over a pool of host memory: a call that raises leaves the cache and the pool as they were."""
import contextlib

import pytest
import torch

from valora_amd import kv_cache
from valora_amd.kv_cache import KVCache


class Pool:
    """What the cache uses of ``MemoryAllocator``."""

    def __init__(self, rows=100, head_num=2, head_dim=64, dtype=torch.float16):
        self.head_num, self.head_dim, self.dtype, self.device, self.tot_size = head_num, head_dim, dtype, torch.device("cpu"), rows
        self.mem_state, self.can_use_mem_size = torch.ones(rows, dtype=torch.bool), rows
        self.key_buffer = torch.empty(1, rows, head_num, head_dim, dtype=dtype)

    def alloc(self, n):
        if n > self.can_use_mem_size:
            raise Exception("no enough pool space")
        rows = torch.nonzero(self.mem_state).flatten()[:n]
        self.mem_state[rows] = False
        self.can_use_mem_size -= n
        return rows

    def free(self, rows):
        self.mem_state[rows] = True
        self.can_use_mem_size += rows.numel()


class Turn:
    """And of ``Rotary``."""

    def __init__(self, head_dim=64):
        self.head_dim, self.freqs = head_dim, torch.zeros(head_dim // 2, dtype=torch.float64)


class Plan:
    def __init__(self, *a, **kw):
        pass


def state(cache):
    return (list(cache.lens), list(cache.seen), cache._changes, cache.mem.can_use_mem_size, cache.mem.mem_state.tolist(), cache.table.tolist())


class Full(torch.Tensor):
    """Rows that cannot be turned into page numbers, as where memory runs out."""

    def to(self, *a, **kw):
        raise torch.OutOfMemoryError("no memory")


@pytest.mark.parametrize("where", ["plan", "rows", "pool"])
def test_a_step_that_raises_changes_nothing(monkeypatch, where):
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    cache = KVCache(Pool(), max_requests=3, max_len=90, q_heads=4, rotary=Turn())
    before_it = cache.step([0, 2], [5, 7])
    before = state(cache)
    with monkeypatch.context() as m:
        if where == "plan":
            def broken(*a, **kw):
                raise torch.OutOfMemoryError("no memory")
            m.setattr(kv_cache, "AttentionPlan", broken)
        elif where == "rows":
            alloc = cache.mem.alloc
            m.setattr(cache.mem, "alloc", lambda n: alloc(n).as_subclass(Full))
            m.setattr(cache.mem, "free", lambda rows: Pool.free(cache.mem, rows.as_subclass(torch.Tensor)))
        with pytest.raises(Exception, match="pool space" if where == "pool" else "no memory"):
            cache.step([2, 1], [1, 88 if where == "pool" else 3])
    assert state(cache) == before and before_it._changes == cache._changes
    # and the same pass again is as if it had not been tried
    step = cache.step([2, 1], [1, 3])
    assert step.positions.tolist() == [7, 0, 1, 2] and step.loc.tolist() == [12, 13, 14, 15]
    assert cache.lens == [5, 3, 8] and cache.mem.can_use_mem_size == 100 - 16
    assert cache.table[1, :4].tolist() == [13, 14, 15, -1] and cache.table[2, 7].item() == 12


def test_heads_that_attention_does_not_take_are_refused_when_the_cache_is_made():
    for pool, kw, message in ((dict(head_dim=80), {}, "head_dim=80"), (dict(head_dim=112), {}, "head_dim=112"), (dict(head_num=3), {}, "multiple of kv_heads=3"),
                              (dict(head_num=8), {}, "multiple of kv_heads=8"), ({}, dict(q_heads=0), "q_heads=0"), ({}, dict(window=-1), "negative"),
                              ({}, dict(max_requests=(1 << 20) + 1), "too large"), (dict(dtype=torch.float32), {}, "dtype=torch.float32")):
        mem = Pool(**pool)
        with pytest.raises(RuntimeError, match=message):
            KVCache(mem, **dict(dict(max_requests=2, max_len=16, q_heads=4, rotary=Turn(mem.head_dim)), **kw))
    far = Turn()
    far.freqs = far.freqs.to("meta")
    with pytest.raises(RuntimeError, match="the rotary is on meta"):
        KVCache(Pool(), 2, 16, 4, far)
    KVCache(Pool(), 0, 0, 4, Turn())


def test_a_slot_that_is_none_is_not_released(monkeypatch):
    """-1 is not the last slot."""
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    cache = KVCache(Pool(), max_requests=3, max_len=90, q_heads=4, rotary=Turn())
    step = cache.step([0, 2], [5, 7])
    before = state(cache)
    for slot in (-1, -3, 3):
        with pytest.raises(RuntimeError, match=rf"slot {slot} is outside \[0, 3\)"):
            cache.release(slot)
    assert state(cache) == before and step._changes == cache._changes


def test_an_eviction_or_release_that_raises_changes_nothing(monkeypatch):
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    cache = KVCache(Pool(), max_requests=2, max_len=20, q_heads=4, rotary=Turn(), track=True)
    step = cache.step([0, 1], [5, 7])
    cache.weights += 1
    before, table, weights = state(cache), cache.table, cache.weights
    monkeypatch.setattr(kv_cache, "evict", lambda t, l, w, *a: (t.clone().fill_(-1), l, torch.zeros_like(w), t.new_full(t.shape, -1).as_subclass(Full)))
    for call in (lambda: cache.evict(4, 2), lambda: cache.release(1)):
        with monkeypatch.context() as m:
            m.setattr(KVCache, "_free", lambda self, rows, count: rows.as_subclass(Full).to(torch.long))
            with pytest.raises(torch.OutOfMemoryError):
                call()
        assert state(cache) == before and step._changes == cache._changes
        assert cache.table is table and cache.weights is weights and bool((weights == 1).all())


def test_the_pool_is_called_with_its_own_device_current(monkeypatch):
    """Another device may be current where the cache is used."""
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    current, calls = [], []

    @contextlib.contextmanager
    def on(device):
        current.append(device)
        yield
        current.pop()

    class Library:
        def mlora_pool_free(self, *a):
            calls.append(("free", list(current)))
            return 0

    cache = KVCache(Pool(), max_requests=2, max_len=20, q_heads=4, rotary=Turn(), track=True)
    alloc = cache.mem.alloc
    monkeypatch.setattr(cache.mem, "alloc", lambda n: (calls.append(("alloc", list(current))), alloc(n))[1])
    monkeypatch.setattr(kv_cache, "_on", on)
    monkeypatch.setattr(kv_cache._lib, "lib", Library)
    monkeypatch.setattr(kv_cache._lib, "current_stream", lambda device: None)
    monkeypatch.setattr(kv_cache, "evict", lambda t, l, w, *a: (t, l, w, t))
    cache.step([0, 1], [5, 7])
    cache.evict(4, 2)
    cache.release(1)
    assert calls == [(name, [torch.device("cpu")]) for name in ("alloc", "free", "free")]
