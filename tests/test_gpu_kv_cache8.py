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


@pytest.mark.parametrize("more", [False, True])
def test_a_layer_over_codes_with_fused_norms(dev, more):
    """Everything together: adapters and the 8-bit cache from one pool, norms fused with the sums at the blocks; a prompt whole and in parts,
    against the layer in 64 bits over the values that the cache holds."""
    import torch.nn.functional as F
    from tests.test_gpu_norm import norm64
    from valora_amd.infer_adapter import InferAdapter, LoraAdapterWeights
    from valora_amd.layer import LayerPlans, LayerPools, LayerWeights, layer_forward
    H, MLP, heads, dtype, r, n = 256, 512, 4, torch.float16, 16, 37
    d = H // heads
    g = torch.Generator().manual_seed(5)
    mem = MemoryAllocator(300, 0, dtype, heads, d, 1, device=dev)
    mem.key_buffer.fill_(math.nan), mem.value_buffer.fill_(math.nan)
    adapters = InferAdapter.init(mem)
    net = {"num_hidden_layers": 1, "hidden_size": H}
    A = [[torch.randn(r, H, generator=g) * 0.05 for _ in range(4)]]
    B = [[torch.randn(H, r, generator=g) * 0.05 for _ in range(4)]]
    adapters.load_adapters([LoraAdapterWeights.from_dense("a", r, 2.0 * r, net, A, B, dtype=dtype, pin=False)])
    mk = lambda i, o: (torch.randn(i, o, generator=g) / i ** 0.5).to(dtype)  # noqa: E731
    vec = lambda: (1 + 0.1 * torch.randn(H, generator=g)).to(dtype)  # noqa: E731
    plain = [mk(H, H), mk(H, H), mk(H, H), mk(H, H), mk(H, MLP), mk(H, MLP), mk(MLP, H), vec(), vec()]
    extra = dict(post1=vec(), post2=vec(), gate1=vec(), gate2=vec(), residual_scale=1.5, block_scale=0.5) if more else {}
    w = LayerWeights(*plain, **extra)
    on = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    wd = LayerWeights(*[on(t) for t in plain], **{k: on(t) for k, t in extra.items()})
    x = torch.randn(n, H, generator=g).to(dtype)
    zero_up = (torch.zeros(64, heads, d, dtype=dtype, device=dev), torch.zeros(64, heads, MLP // heads, dtype=dtype, device=dev))

    def forward(cache, rows, slot):
        step = cache.step([slot], [rows.shape[0]])
        ids = torch.zeros(rows.shape[0], dtype=torch.long, device=dev)
        pools = LayerPools((mem.key_buffer[0], mem.value_buffer[0]), zero_up, (zero_up[1], zero_up[0]), adapters.a_start, adapters.a_len,
                           adapters.a_loc, adapters.a_scaling)
        plans = LayerPlans(ids, adapters.a_start, adapters.a_len, r, H, MLP)
        return layer_forward(rows, wd, pools, plans, step.attention(0), heads, fused=True)

    assert int(adapters.a_loc.max()) < 64                # (the rows the zero buffers are indexed with)
    before = mem.key_buffer[0][adapters.a_loc].clone()
    cache = KVCache(mem, max_requests=2, max_len=63, q_heads=heads, rotary=Rotary(d, device=dev), codes=True)
    whole = forward(cache, x.to(dev), 0)
    parts = torch.cat([forward(cache, x[a:b].to(dev), 1) for a, b in ((0, 19), (19, 20), (20, 36), (36, 37))])
    torch.cuda.synchronize()
    assert torch.equal(mem.key_buffer[0][adapters.a_loc], before)

    eff = lambda base, s: base.double() + 2.0 * A[0][s].to(dtype).double().T @ B[0][s].to(dtype).double().T  # noqa: E731
    n64 = lambda z, wt: z if wt is None else norm64(z, wt, None, 1e-6, "rms", 0.0)  # noqa: E731
    one = lambda t: 1.0 if t is None else t.double()  # noqa: E731
    h = n64(x.double(), w.ln1)
    q, k, v = ((h @ eff(m, s)).view(n, heads, d) for s, m in enumerate((w.wq, w.wk, w.wv)))
    q, k = rotate(q, torch.arange(n), d), rotate(k, torch.arange(n), d)
    for slot, got in ((0, whole), (1, parts)):
        kc, vc = (t.cpu().double() for t in cache.read(slot, 0))
        # half a step of a code, of a value that is off by some roundings of 2^-11 of its sums: 2^-8 of the largest
        for mine, exact in ((kc, k), (vc, v)):
            assert bool(((mine - exact).abs() <= exact.abs() * 2.0 ** -4 + 2.0 ** -8 * exact.abs().amax(-1, keepdim=True)).all())
        a = torch.empty(n, heads, d, dtype=torch.float64)
        for i in range(heads):
            s = (q[:, i] @ kc[:, i].T * d ** -0.5).masked_fill(torch.ones(n, n).tril() == 0, -math.inf)
            a[:, i] = torch.softmax(s, -1) @ vc[:, i]
        y = w.residual_scale * x.double() + w.block_scale * one(w.gate1) * n64(a.view(n, H) @ eff(w.wo, 3), w.post1)
        h2 = n64(y, w.ln2)
        want = w.residual_scale * y + w.block_scale * one(w.gate2) * n64((F.silu(h2 @ w.w_gate.double()) * (h2 @ w.w_up.double())) @ w.w_down.double(), w.post2)
        # about a dozen roundings of 2^-12 of the values on the way, of which few reach the output whole
        err = float((got.cpu().double() - want).norm() / want.norm())
        assert err <= 12 * 2.0 ** -12, (slot, err)
