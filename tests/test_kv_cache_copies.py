"""What a step of the cache sends to the device, without a GPU: as few copies in 8 bits as in 16."""
import pytest
import torch

from tests.test_kv_cache_step import Plan, Pool, Turn
from valora_amd import kv_cache
from valora_amd.kv_cache import KVCache


@pytest.mark.parametrize("codes", [False, True])
def test_copies_of_a_step(monkeypatch, codes):
    """The places of its tokens in one, the plan's lengths in another."""
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    cache = KVCache(Pool(), max_requests=3, max_len=90, q_heads=4, rotary=Turn(), codes=codes)
    made, tensor = [], torch.tensor
    monkeypatch.setattr(torch, "tensor", lambda *a, **kw: (made.append(kw.get("dtype")), tensor(*a, **kw))[1])
    for slots, lens in (([0, 2], [5, 7]), ([2, 0], [1, 1]), ([1], [3])):
        made.clear()
        cache.step(slots, lens)
        assert sorted(made, key=str) == [torch.int32, torch.long]


@pytest.mark.parametrize("page", [2, 4])
def test_places_against_a_list(monkeypatch, page):
    """Random passes against a table kept by hand: every token's slot is the one that its row and place in it give, rows are taken once."""
    monkeypatch.setattr(kv_cache, "AttentionPlan", Plan)
    cache = KVCache(Pool(rows=400), max_requests=5, max_len=150, q_heads=4, rotary=Turn(), codes=True)
    cache.page = page
    g = torch.Generator().manual_seed(page)
    tokens = [[] for _ in range(5)]                       # each slot's tokens' places
    for _ in range(40):
        slots = torch.randperm(5, generator=g)[:int(torch.randint(1, 6, (1,), generator=g))].tolist()
        lens = [int(torch.randint(1, 8, (1,), generator=g)) for _ in slots]
        if any(cache.lens[s] + n > 75 for s, n in zip(slots, lens)):
            cache.lens, cache.seen, tokens = [0] * 5, [0] * 5, [[] for _ in range(5)]
            cache.table.fill_(-1)
            cache.mem.mem_state.fill_(True)
            cache.mem.can_use_mem_size = 400
        step = cache.step(slots, lens)
        at = 0
        for s, n in zip(slots, lens):
            first = len(tokens[s])
            assert step.positions[at:at + n].tolist() == list(range(first, first + n))
            tokens[s] += step.loc[at:at + n].tolist()
            at += n
            rows = cache.table[s].tolist()
            assert tokens[s] == [rows[j // page] * page + j % page for j in range(len(tokens[s]))]
            assert all(r >= 0 for r in rows[:-(-len(tokens[s]) // page)]) and rows[-(-len(tokens[s]) // page)] == -1
        held = [r for row in cache.table.tolist() for r in row if r >= 0]
        assert len(set(held)) == len(held) == 400 - cache.mem.can_use_mem_size
