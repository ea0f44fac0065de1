"""GPU: the cache of 8-bit codes as a serving loop uses it: prompts in chunks and decode steps over rows of one pool, two tokens a row, through
the rotation, the codes and the attention over them; eviction by rows, reading back, rows given back; a captured step."""
import math

import pytest
import torch

from tests._cache8 import decode, encode
from tests.test_gpu_kv_cache import Dense, rotate
from valora_amd.infer_adapter import MemoryAllocator
from valora_amd.kv_cache import KVCache
from valora_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


class Coded(Dense):
    """A request's cache and its attention from the definition, 64 bits: k and v as their codes stand for them."""

    def attend(self, q, k, v, first):
        pos = torch.arange(first, first + q.shape[0])
        self.new = rotate(k.double(), pos, self.d)
        values = decode(*encode(self.new, self.dtype))
        q = rotate(q.double(), pos, self.d).to(self.dtype).double()
        self.k = values if self.k is None else torch.cat([self.k, values])
        v = decode(*encode(v, self.dtype))
        self.v = v if self.v is None else torch.cat([self.v, v])
        n, length, group = q.shape[0], self.k.shape[0], q.shape[1] // self.k.shape[1]
        old = torch.zeros(0, dtype=torch.float64) if self.weight is None else self.weight
        self.weight = torch.cat([old, torch.zeros(n, dtype=torch.float64)])
        sees = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
        out = torch.empty_like(q)
        for h in range(q.shape[1]):
            s = (q[:, h] @ self.k[:, h // group].T * self.d ** -0.5).masked_fill(~sees, -math.inf)
            p = torch.softmax(s, -1)
            out[:, h] = p @ self.v[:, h // group]
            self.weight += p.sum(0)
        return out


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float16, 4, 2, 64), (torch.bfloat16, 8, 1, 128), (torch.bfloat16, 3, 3, 96)])
def test_prompts_decoding_eviction_and_release(dev, dtype, hq, hkv, d):
    g = torch.Generator().manual_seed(1)
    mem = MemoryAllocator(400, 0, dtype, hkv, d, 2, device=dev)
    mem.key_buffer.fill_(math.nan)
    mem.value_buffer.fill_(math.nan)                     # rows that were never written
    cache = KVCache(mem, max_requests=4, max_len=301, q_heads=hq, rotary=Rotary(d, device=dev), track=True, codes=True)
    dense, seen = {}, {}
    u = torch.finfo(dtype).eps / 2

    def step(slots, lens):
        T = sum(lens)
        q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
        s = cache.step(slots, lens)
        got = s.attention(1)(q.view(T, -1).to(dev), k.view(T, -1).to(dev), v.view(T, -1).to(dev))
        torch.cuda.synchronize()
        at = 0
        for slot, n in zip(slots, lens):
            c = dense.setdefault(slot, Coded(d, dtype))
            want = c.attend(q[at:at + n], k[at:at + n], v[at:at + n], seen.get(slot, 0))
            seen[slot] = seen.get(slot, 0) + n
            # The rotated q of a few elements may round the other way (a score then moves by 2 u of one product of d), the weights of the
            # second product are rounded, the result is rounded: 4 u of the largest value covers each
            room = 3 * 4 * u * float(c.v.abs().max())
            err = float((got[at:at + n].view(n, hq, d).cpu().double() - want).abs().max())
            assert err <= room, (slot, err, room)
            at += n

    def check_rows():
        state = mem.mem_state.cpu()
        used = torch.cat([cache.table[s, :-(-cache.lens[s] // 2)].cpu().long() for s in range(4)])
        assert len(set(used.tolist())) == len(used) and int(state.sum()) == mem.can_use_mem_size == free - len(used) and not state[used].any()

    free = mem.can_use_mem_size
    step([2, 0], [90, 41])
    step([0, 2, 1], [1, 31, 150])
    for _ in range(5):
        step([1, 0, 2], [1, 1, 1])
    assert cache.lens == [47, 155, 126, 0]
    check_rows()
    for slot in (0, 1, 2):
        assert torch.allclose(cache.weights[slot, :cache.lens[slot]].cpu().double(), dense[slot].weight, rtol=2e-2, atol=2e-2)
        k, v = cache.read(slot, 1)                       # (a key's code next to a border may be the neighbour: the sines are the device's)
        assert torch.equal(v.cpu().double(), dense[slot].v)
        assert float((k.cpu().double() != dense[slot].k).double().mean()) <= 1e-3
    assert cache.read(3, 1)[0].shape == (0, hkv, d)
    w, before = cache.weights.cpu(), cache.table.cpu()
    # 65 tokens are 32 rows; 9 recent ones 5 rows, 1 first one a row
    assert cache.evict(budget=65, recent=9, sinks=1) == (78 - 32) + (63 - 32)
    assert cache.lens == [47, 155 - 2 * 46, 126 - 2 * 31, 0]
    check_rows()
    for slot in (1, 2):
        n = len(dense[slot].weight)
        rows = -(-n // 2)
        mass = torch.cat([w[slot, :n], torch.zeros(n % 2)]).view(rows, 2).sum(1)
        middle = torch.sort(mass[1:rows - 5], descending=True, stable=True).indices[:26] + 1
        stay = torch.cat([torch.arange(1), middle.sort().values, torch.arange(rows - 5, rows)])
        dense[slot].keep((stay[:, None] * 2 + torch.arange(2)).flatten()[:cache.lens[slot]])
        assert torch.equal(cache.table[slot, :32].cpu(), before[slot, stay]) and bool((cache.table[slot, 32:] == -1).all())
    for _ in range(3):                                   # positions go on from where they were, odd lengths from their half row
        step([2, 1, 0], [1, 2, 1])
    check_rows()
    cache.release(1)
    dense.pop(1), seen.pop(1)
    step([3, 1], [20, 5])
    check_rows()
    empty = cache.step([], [])
    assert empty.attention(0)(*(torch.empty(0, h * d, dtype=dtype, device=dev) for h in (hq, hkv, hkv))).shape == (0, hq * d)
    for slot in range(4):
        cache.release(slot)
    assert mem.can_use_mem_size == free and int(mem.mem_state.sum()) == free and not cache.weights.any()


def test_read_of_a_cache_in_16_bits(dev):
    mem = MemoryAllocator(50, 0, torch.float16, 2, 64, 1, device=dev)
    cache = KVCache(mem, 2, 16, 4, Rotary(64, device=dev))
    x = torch.randn(5, 384, dtype=torch.float16, device=dev)
    cache.step([1], [5]).attention(0)(x[:, :256], x[:, :128], x[:, 128:256])
    k, v = cache.read(1, 0)
    assert torch.equal(v, x[:, 128:256].reshape(5, 2, 64)) and torch.equal(k[0], x[0, :128].view(2, 64))
    with pytest.raises(RuntimeError, match="slot -1"):
        cache.read(-1, 0)


def test_a_captured_decode_step(dev):
    """Storing, attention and reading back in one graph, replayed over changing tokens, slots and lengths between eager calls of the same
    operators; every replay against the eager result."""
    from valora_amd import cache8
    from valora_amd.attention import AttentionPlan
    g = torch.Generator(device="cpu").manual_seed(2)
    hq, hk, d, page, B, rows = 8, 2, 64, 4, 3, 60
    dtype = torch.bfloat16
    rotary = Rotary(d, device=dev)
    kc, vc = (torch.zeros(rows, hk, page, d, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    powers = cache8.new_powers((rows, hk, page), dev)
    table = torch.randperm(rows, generator=g)[:B * 20].view(B, 20).to(torch.int32).to(dev)
    q, k, v = (torch.zeros(B, h, d, dtype=dtype, device=dev) for h in (hq, hk, hk))
    positions, loc = torch.zeros(B, dtype=torch.long, device=dev), torch.zeros(B, dtype=torch.long, device=dev)
    start, one, kv = (torch.tensor(t, dtype=torch.int32, device=dev) for t in ([0, 1, 2], [1, 1, 1], [1, 1, 1]))
    turned, out = torch.empty_like(q), torch.empty_like(q)
    plan = AttentionPlan(start, one, kv, n_tokens=B, max_seq_len=1, max_kv_len=80, q_heads=hq, kv_heads=hk, head_dim=d, page_size=page)

    def step():
        plan.rebuild()
        rotary.store8(positions, q, k, v, kc, vc, powers, loc, q_out=turned)
        plan.attend8(out, turned, kc, vc, powers, table)
        return cache8.read(kc, vc, powers, loc, dtype)

    def fill(n, seed):
        h = torch.Generator().manual_seed(seed)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=h).to(dtype))
        positions.fill_(n)
        kv.fill_(n + 1)
        loc.copy_(table[:, n // page].long() * page + n % page)

    fill(0, 0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        back = step()
    for n in range(1, 9):
        fill(n * 9, n)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got, got_back = out.clone(), [t.clone() for t in back]
        out.fill_(3.0)
        again = step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and all(torch.equal(a, b) for a, b in zip(got_back, again))
        assert float(got.abs().max()) < 7.0


def test_another_stream(dev):
    g = torch.Generator().manual_seed(3)
    mem = MemoryAllocator(60, 0, torch.float16, 2, 64, 1, device=dev)
    x = torch.randn(40, 512, generator=g).to(torch.float16).to(dev)
    results = []
    for stream in (torch.cuda.current_stream(dev), torch.cuda.Stream(dev)):
        stream.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(stream):
            cache = KVCache(mem, 1, 64, 4, Rotary(64, device=dev), codes=True)
            results.append(cache.step([0], [40]).attention(0)(x[:, :256], x[:, 256:384], x[:, 384:]))
            cache.release(0)
        stream.synchronize()
    assert torch.equal(*results)
