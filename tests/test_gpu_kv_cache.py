"""GPU: the cache's operators together, as a serving loop uses them: prompts in chunks and decode steps of several requests over one
pool that adapters share, through ``layer_forward``; eviction and the steps after it; rows given back."""
import math

import pytest
import torch
import torch.nn.functional as F

from valora_amd import workloads as W
from valora_amd.infer_adapter import InferAdapter, LoraAdapterWeights, MemoryAllocator
from valora_amd.kv_cache import KVCache
from valora_amd.layer import LayerPlans, LayerPools, LayerWeights, layer_forward, rmsnorm
from valora_amd.rotary import Rotary, frequencies

pytestmark = pytest.mark.gpu


def rotate(x, positions, d):
    radians, _ = frequencies(d)
    angle = positions.double()[:, None] * torch.tensor(radians, dtype=torch.float64)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


class Dense:
    """A request's cache and its attention from the definition, 64 bits: k and v as they were rounded when they were stored."""

    def __init__(self, d, dtype):
        self.d, self.dtype = d, dtype
        self.k, self.v, self.weight = None, None, None

    def attend(self, q, k, v, first):
        n = q.shape[0]
        pos = torch.arange(first, first + n)
        q, k = (rotate(t.double(), pos, self.d).to(self.dtype).double() for t in (q, k))
        self.k = k if self.k is None else torch.cat([self.k, k])
        self.v = v.double() if self.v is None else torch.cat([self.v, v.double()])
        old = torch.zeros(0, dtype=torch.float64) if self.weight is None else self.weight
        self.weight = torch.cat([old, torch.zeros(n, dtype=torch.float64)])
        length, group = self.k.shape[0], q.shape[1] // self.k.shape[1]
        sees = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
        out = torch.empty_like(q)
        for h in range(q.shape[1]):
            s = (q[:, h] @ self.k[:, h // group].T * self.d ** -0.5).masked_fill(~sees, -math.inf)
            p = torch.softmax(s, -1)
            out[:, h] = p @ self.v[:, h // group]
            self.weight += p.sum(0)
        return out

    def keep(self, stay):
        self.k, self.v, self.weight = self.k[stay], self.v[stay], self.weight[stay]


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float16, 4, 2, 64), (torch.bfloat16, 8, 1, 128)])
def test_prompts_decoding_eviction_and_release(dev, dtype, hq, hkv, d):
    g = torch.Generator().manual_seed(1)
    mem = MemoryAllocator(700, 0, dtype, hkv, d, 1, device=dev)
    mem.key_buffer.fill_(math.nan)
    mem.value_buffer.fill_(math.nan)                     # rows that were never written
    cache = KVCache(mem, max_requests=4, max_len=300, q_heads=hq, rotary=Rotary(d, device=dev), track=True)
    dense, seen = {}, {}
    u = torch.finfo(dtype).eps / 2

    def step(slots, lens):
        T = sum(lens)
        q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
        s = cache.step(slots, lens)
        got = s.attention(0)(q.view(T, -1).to(dev), k.view(T, -1).to(dev), v.view(T, -1).to(dev))
        torch.cuda.synchronize()
        at = 0
        for slot, n in zip(slots, lens):
            c = dense.setdefault(slot, Dense(d, dtype))
            want = c.attend(q[at:at + n], k[at:at + n], v[at:at + n], seen.get(slot, 0))
            seen[slot] = seen.get(slot, 0) + n
            # The rotated q and k of a few elements may round the other way (a score then moves by 2 u of one product of d), the
            # weights of the second product are rounded, the result is rounded: 4 u of the largest value covers each
            room = 4 * 4 * u * float(c.v.abs().max())
            err = float((got[at:at + n].view(n, hq, d).cpu().double() - want).abs().max())
            assert err <= room, (slot, err, room)
            at += n

    free = mem.can_use_mem_size
    step([2, 0], [90, 40])
    step([0, 2, 1], [1, 30, 150])
    for _ in range(5):
        step([1, 0, 2], [1, 1, 1])
    assert cache.lens == [46, 155, 125, 0] and mem.can_use_mem_size == free - 326
    for slot in (0, 1, 2):
        assert torch.allclose(cache.weights[slot, :cache.lens[slot]].cpu().double(), dense[slot].weight, rtol=2e-2, atol=2e-2)
    # eviction: what goes is decided by the weights on the device
    w = cache.weights.cpu()
    before = cache.table.cpu()
    assert cache.evict(budget=64, recent=10, sinks=2) == (155 - 64) + (125 - 64)
    assert cache.lens == [46, 64, 64, 0] and mem.can_use_mem_size == free - 174
    for slot in (1, 2):
        n = len(dense[slot].weight)
        middle = torch.sort(w[slot, 2:n - 10], descending=True, stable=True).indices[:52] + 2
        stay = torch.cat([torch.arange(2), middle.sort().values, torch.arange(n - 10, n)])
        dense[slot].keep(stay)
        assert torch.equal(cache.table[slot, :64].cpu(), before[slot, stay]) and bool((cache.table[slot, 64:] == -1).all())
        assert torch.equal(cache.weights[slot, :64].cpu(), w[slot, stay]) and not cache.weights[slot, 64:].any()
    state = mem.mem_state.cpu()
    used = torch.cat([cache.table[s, :cache.lens[s]].cpu().long() for s in range(4)])
    assert int(state.sum()) == mem.can_use_mem_size and not state[used].any()
    for _ in range(3):                                   # positions go on from where they were
        step([2, 1, 0], [1, 2, 1])
    cache.release(1)
    dense.pop(1), seen.pop(1)
    step([3, 1], [20, 5])                                # rows and slot are used again
    empty = cache.step([], [])                           # a pass without tokens
    assert empty.attention(0)(*(torch.empty(0, h * d, dtype=dtype, device=dev) for h in (hq, hkv, hkv))).shape == (0, hq * d)
    cache.release(0), cache.release(1), cache.release(2), cache.release(3)
    assert mem.can_use_mem_size == free and int(mem.mem_state.sum()) == free and not cache.weights.any()


def test_a_layer_with_adapters_and_cache_from_one_pool(dev):
    """Adapter rows and cached tokens come from one allocator; ``layer_forward`` decodes a prompt token by token and gives what one
    pass over the whole prompt gives, and both what the layer gives in 32 bits with dense effective weights."""
    H, MLP, heads, dtype, r = 256, 512, 4, torch.float16, 16
    d = H // heads
    g = torch.Generator().manual_seed(2)
    mem = MemoryAllocator(400, 0, dtype, heads, d, 1, device=dev)
    mem.key_buffer.fill_(math.nan), mem.value_buffer.fill_(math.nan)
    adapters = InferAdapter.init(mem)
    net = {"num_hidden_layers": 1, "hidden_size": H}
    A = [[torch.randn(r, H, generator=g) * 0.05 for _ in range(4)]]
    B = [[torch.randn(H, r, generator=g) * 0.05 for _ in range(4)]]
    adapters.load_adapters([LoraAdapterWeights.from_dense("a", r, 2.0 * r, net, A, B, dtype=dtype, pin=False)])
    mk = lambda i, o: (torch.randn(i, o, generator=g) / i ** 0.5).to(dtype)  # noqa: E731
    w = LayerWeights(mk(H, H), mk(H, H), mk(H, H), mk(H, H), mk(H, MLP), mk(H, MLP), mk(MLP, H),
                     (1 + 0.1 * torch.randn(H, generator=g)).to(dtype), (1 + 0.1 * torch.randn(H, generator=g)).to(dtype))
    wd = LayerWeights(*[getattr(w, f).to(dev) for f in ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down", "ln1", "ln2")])
    n = 37
    x = torch.randn(n, H, generator=g).to(dtype)
    # the attention projections' adapter, and no adapter on the others (their slots hold zeros)
    zero_up = (torch.zeros(64, heads, d, dtype=dtype, device=dev), torch.zeros(64, heads, MLP // heads, dtype=dtype, device=dev))
    zero_down = (zero_up[1], zero_up[0])

    def forward(cache, rows, slot):
        step = cache.step([slot], [rows.shape[0]])
        ids = torch.zeros(rows.shape[0], dtype=torch.long, device=dev)
        loc = adapters.a_loc
        pools = LayerPools((mem.key_buffer[0], mem.value_buffer[0]), zero_up, zero_down, adapters.a_start, adapters.a_len, loc, adapters.a_scaling)
        plans = LayerPlans(ids, adapters.a_start, adapters.a_len, r, H, MLP)
        return layer_forward(rows, wd, pools, plans, step.attention(0), heads)

    assert int(adapters.a_loc.max()) < 64                # (the rows the zero buffers are indexed with)
    cache = KVCache(mem, max_requests=2, max_len=64, q_heads=heads, rotary=Rotary(d, device=dev))
    whole = forward(cache, x.to(dev), 0)
    parts = torch.cat([forward(cache, x[a:b].to(dev), 1) for a, b in ((0, 20), (20, 21), (21, 36), (36, 37))])
    torch.cuda.synchronize()

    xf = x.double()
    eff = lambda base, s: base.double() + 2.0 * A[0][s].to(dtype).double().T @ B[0][s].to(dtype).double().T  # noqa: E731
    h = rmsnorm(x.float(), w.ln1.float()).double()
    q, k, v = (h @ eff(m, s) for s, m in enumerate((w.wq, w.wk, w.wv)))
    c = Dense(d, torch.float64)
    a = c.attend(q.view(n, heads, d), k.view(n, heads, d), v.view(n, heads, d), 0).view(n, H)
    y = xf + a @ eff(w.wo, 3)
    h2 = rmsnorm(y.float(), w.ln2.float()).double()
    want = y + (F.silu(h2 @ w.w_gate.double()) * (h2 @ w.w_up.double())) @ w.w_down.double()
    rel = lambda p: float((p.cpu().double() - want).norm() / want.norm())  # noqa: E731
    # about a dozen roundings of 2^-12 of the values on the way, of which few reach the output whole
    assert rel(whole) <= 12 * 2.0 ** -12, rel(whole)
    assert rel(parts) <= 12 * 2.0 ** -12, rel(parts)


def test_refusals(dev):
    mem = MemoryAllocator(20, 0, torch.float16, 2, 64, 1, device=dev)
    with pytest.raises(RuntimeError, match="head_dim"):
        KVCache(mem, 2, 16, 4, Rotary(32, device=dev))
    cache = KVCache(mem, 2, 16, 4, Rotary(64, device=dev))
    for slots, lens, message in (([0, 0], [1, 1], "distinct"), ([2], [1], "outside"), ([0], [0], "new tokens"), ([0], [17], "max_len"), ([0, 1], [3], "distinct")):
        with pytest.raises(RuntimeError, match=message):
            cache.step(slots, lens)
    cache.step([0], [16])
    with pytest.raises(Exception, match="no enough pool space"):
        cache.step([1], [5])
    assert cache.lens == [16, 0] and mem.can_use_mem_size == 4
    with pytest.raises(RuntimeError, match="track"):
        cache.evict(4, 1)
    tracked = KVCache(mem, 1, 4, 4, Rotary(64, device=dev), window=8, track=True)
    with pytest.raises(RuntimeError, match="window"):
        tracked.evict(4, 1)
    old = cache.step([1], [2])
    cache.step([1], [1])
    x = torch.zeros(2, 256, dtype=torch.float16, device=dev)
    with pytest.raises(RuntimeError, match="changed"):
        old.attention(0)(x, x[:, :128], x[:, :128])
