"""GPU: the norms around a block against their definition in 64 bits."""
import pytest
import torch

from valora_amd.norm import block_norm

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def norm64(z, w, b, eps, kind, offset):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    y = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * (offset + w.double())
    return y if b is None else y + b.double()


def definition(x, weight, bias, block, block_weight, block_bias, gate, a, s, eps, kind, offset):
    """(r, h) and what each may be off by before its rounding.  Sums of H products in 32 bits, in a tree of at most 64 + 16 + 64 terms in a
    row: (80 + 16) * 2^-24 relative to the sum of sizes is above it; a norm's factor takes half of that and a handful of roundings."""
    u = 2.0 ** -24
    x = x.double()
    r = x
    off = torch.zeros_like(x)
    if block is not None:
        o, g = block.double(), 1.0 if gate is None else gate.double()
        o_off = torch.zeros_like(o)
        if block_weight is not None:
            n = norm64(o, block_weight, block_bias, eps, kind, offset)
            spread = (o - (o.mean(-1, keepdim=True) if kind == "layer" else 0)).abs() + (o.abs().mean(-1, keepdim=True) if kind == "layer" else 0)
            scale = (offset + block_weight.double()).abs() / torch.sqrt(((o - (o.mean(-1, keepdim=True) if kind == "layer" else 0)) ** 2).mean(-1, keepdim=True) + eps)
            o_off = 128 * u * spread * scale + 4 * u * n.abs()
            o = n
        a32, s32 = float(torch.tensor(a)), float(torch.tensor(s))
        r = a32 * x + s32 * g * o
        off = abs(s32) * (g if isinstance(g, float) else g.abs()) * (o_off + 4 * u * o.abs()) + 4 * u * (a32 * x).abs()
    h = h_off = None
    if weight is not None:
        h = norm64(r, weight, bias, eps, kind, offset)
        c = r - (r.mean(-1, keepdim=True) if kind == "layer" else 0)
        size = r.abs() + (r.abs().mean(-1, keepdim=True) if kind == "layer" else 0)
        root = torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        scale = (offset + weight.double()).abs() / root
        # r's own error moves the row's root by at most its own, relative to it
        h_off = scale * (off + 128 * u * size + c.abs() * (off.abs().amax(-1, keepdim=True) / root + 128 * u)) + 8 * u * h.abs()
        if kind == "layer":
            h_off = h_off + scale * off.mean(-1, keepdim=True)
        if bias is not None:
            h_off = h_off + 2 * u * bias.double().abs()
    return r, off, h, h_off


def close(got, want, off, dtype):
    least = {F16: 2.0 ** -25, BF16: 2.0 ** -134}[dtype]
    over = (got.cpu().double() - want).abs() - (want.abs() + off) * torch.finfo(dtype).eps / 2 - off - least
    assert bool((over <= 0).all()), (float(over.max()), torch.nonzero(over > 0)[:3].tolist())


def case(dtype, T, H, kind, block, post, gate, bias, param=None, seed=0, mean=0.0):
    g = torch.Generator().manual_seed(seed + T * 31 + H)
    param = dtype if param is None else param
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (rnd(T, H) + mean)
    x[:, ::97] *= 20
    c = dict(x=x.to(dtype), weight=(1 + 0.2 * rnd(H)).to(param), bias=(0.1 * rnd(H)).to(param) if bias else None)
    c["block"] = (0.7 * rnd(T, H)).to(dtype) if block else None
    c["block_weight"] = (1 + 0.2 * rnd(H)).to(param) if post else None
    c["block_bias"] = (0.1 * rnd(H)).to(param) if post and bias else None
    c["gate"] = {None: None, "channel": rnd(H).to(param), "token": rnd(T, 1).to(param), "element": rnd(T, H).to(param)}[gate]
    return c


def check(dev, c, a=1.0, s=1.0, eps=1e-6, kind="rms", offset=0.0, **kw):
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    r, h = block_norm(to(c["x"]), to(c["weight"]), to(c["bias"]), block=to(c["block"]), block_weight=to(c["block_weight"]),
                      block_bias=to(c["block_bias"]), gate=to(c["gate"]), residual_scale=a, block_scale=s, eps=eps, kind=kind, offset=offset, **kw)
    want = definition(c["x"], c["weight"], c["bias"], c["block"], c["block_weight"], c["block_bias"], c["gate"], a, s,
                      float(torch.tensor(eps)), kind, offset)
    dtype = c["x"].dtype
    if c["block"] is None:
        assert torch.equal(r.cpu(), c["x"])
    else:
        close(r, want[0], want[1], dtype)
    if c["weight"] is not None:
        close(h, want[2], want[3], dtype)
    return r, h


WIDTHS = [1, 2, 7, 8, 9, 64, 96, 511, 512, 513, 1000, 1024, 1032, 2048, 4096, 4104, 5120, 8192, 8200, 11008, 16384, 20000, 20001, 32761, 32768]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H", WIDTHS)
def test_widths(dev, dtype, H):
    for T in (1, 5):
        check(dev, case(dtype, T, H, "rms", True, False, None, False))
        check(dev, case(dtype, T, H, "layer", True, True, "channel", True), a=1.5, s=0.25, kind="layer")
        check(dev, case(dtype, T, H, "rms", False, False, None, True))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "token", "element"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_forms(dev, dtype, kind, post, gate, bias, f32):
    for T, H in ((3, 768), (70, 130), (600, 1024)):
        c = case(dtype, T, H, kind, True, post, gate, bias, torch.float32 if f32 else None)
        check(dev, c, a=0.7, s=1.3, eps=1e-5, kind=kind, offset=1.0 if post else 0.0)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_mean_far_from_zero_and_rows_alike(dev, kind):
    """A variance far below the mean's square is that of the differences; rows all of whose elements are alike have none."""
    check(dev, case(BF16, 4, 4096, kind, False, False, None, True, mean=100.0), kind=kind)
    c = case(F16, 3, 640, kind, False, False, None, False)
    c["x"][0], c["x"][1], c["x"][2] = 0.0, 3.0, -60000.0
    check(dev, c, kind=kind, eps=1e-3)


def test_no_norm_after_the_sum(dev):
    c = case(BF16, 9, 300, "rms", True, True, "token", False)
    c["weight"] = None
    r, h = check(dev, c)
    assert h is None


def test_in_place_and_strides(dev):
    c = case(F16, 33, 520, "rms", True, True, "element", False)
    x, block = c["x"].to(dev), c["block"].to(dev)
    r0, h0 = check(dev, c)
    args = dict(block_weight=c["block_weight"].to(dev), gate=c["gate"].to(dev))
    r, h = block_norm(x, c["weight"].to(dev), block=block, residual_out=x, out=block, **args)
    assert r.data_ptr() == x.data_ptr() and torch.equal(r, r0) and torch.equal(h, h0)
    # rows apart, not at 16 bytes
    for gap in (8, 3):
        wide = torch.full((33, 520 + gap), 5.0, dtype=F16, device=dev)
        xs, bs, ro, ho = (wide.clone()[:, gap:] for _ in range(4))
        xs.copy_(c["x"]), bs.copy_(c["block"])
        r, h = block_norm(xs, c["weight"].to(dev), block=bs, residual_out=ro, out=ho, **args)
        close(r, r0.cpu().double(), r0.cpu().double().abs() * 2.0 ** -10, F16)
        close(h, h0.cpu().double(), h0.cpu().double().abs() * 2.0 ** -10, F16)
        assert bool((ro._base[:, :gap] == 5.0).all()) and bool((ho._base[:, :gap] == 5.0).all())


def test_values_that_are_no_numbers_stay_in_their_row(dev):
    c = case(BF16, 6, 256, "rms", True, True, None, False)
    clean = check(dev, c)
    x, block = c["x"].clone(), c["block"].clone()
    x[1, 3], block[4, 9] = float("nan"), float("inf")
    r, h = block_norm(x.to(dev), c["weight"].to(dev), block=block.to(dev), block_weight=c["block_weight"].to(dev))
    for i in (0, 2, 3, 5):
        assert torch.equal(r[i], clean[0][i]) and torch.equal(h[i], clean[1][i])
    assert bool(torch.isnan(h[1]).all()) and bool(torch.isnan(r[1, 3])) and bool(torch.isnan(h[4]).any())


def test_nothing_to_do(dev):
    x = torch.empty(0, 64, dtype=F16, device=dev)
    r, h = block_norm(x, torch.ones(64, dtype=F16, device=dev), block=torch.empty_like(x))
    assert r.shape == h.shape == (0, 64)


def test_layer_forward_with_fused_norms(dev):
    """One decoder layer, its norms fused: plain, and with norms after its blocks, gates and scales, against the layer in 64 bits."""
    import torch.nn.functional as F
    from valora_amd.layer import LayerWeights, layer_forward, segment_attention
    H, MLP, heads, T, dtype = 256, 512, 4, 37, BF16
    g = torch.Generator().manual_seed(6)
    mk = lambda i, o: (torch.randn(i, o, generator=g) / i ** 0.5).to(dtype)  # noqa: E731
    vec = lambda: (1 + 0.1 * torch.randn(H, generator=g)).to(dtype)  # noqa: E731
    plain = [mk(H, H), mk(H, H), mk(H, H), mk(H, H), mk(H, MLP), mk(H, MLP), mk(MLP, H), vec(), vec()]
    more = dict(post1=vec(), post2=vec(), gate1=vec(), gate2=vec(), residual_scale=1.25, block_scale=0.5)
    x = torch.randn(T, H, generator=g).to(dtype)
    on = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731

    def layer64(w):
        n64 = lambda z, wt: z if wt is None else norm64(z, wt, None, 1e-6, "rms", 0.0)  # noqa: E731
        one = lambda t: 1.0 if t is None else t.double()  # noqa: E731
        xd, m = x.double(), [t.double() for t in plain]
        h = n64(xd, w.ln1)
        q, k, v = ((h @ m[i]).view(T, heads, -1).transpose(0, 1) for i in range(3))
        a = F.scaled_dot_product_attention(q[None], k[None], v[None], is_causal=True)[0].transpose(0, 1).reshape(T, H)
        y = w.residual_scale * xd + w.block_scale * one(w.gate1) * n64(a @ m[3], w.post1)
        h2 = n64(y, w.ln2)
        return w.residual_scale * y + w.block_scale * one(w.gate2) * n64((F.silu(h2 @ m[4]) * (h2 @ m[5])) @ m[6], w.post2)

    for extra in ({}, more):
        w = LayerWeights(*plain, **extra)
        wd = LayerWeights(*[on(t) for t in plain], **{k: on(t) for k, t in extra.items()})
        got = layer_forward(x.to(dev), wd, None, None, segment_attention([T], heads), heads, fused=True)
        want = layer64(w)
        # about a dozen roundings of 2^-9 of the values on the way, of which few reach the output whole
        assert float((got.cpu().double() - want).norm() / want.norm()) <= 12 * 2.0 ** -9
        if extra:
            with pytest.raises(RuntimeError, match="fused=True"):
                layer_forward(x.to(dev), wd, None, None, segment_attention([T], heads), heads)


def test_replays_of_a_captured_norm(dev):
    c = case(F16, 12, 640, "rms", True, True, "token", False)
    x, block, w = c["x"].to(dev), c["block"].to(dev), c["weight"].to(dev)
    args = dict(block=block, block_weight=c["block_weight"].to(dev), gate=c["gate"].to(dev))
    block_norm(x, w, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, h = block_norm(x, w, **args)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).to(F16))
        graph.replay()
        torch.cuda.synchronize()
        again = block_norm(x, w, **args)
        assert torch.equal(r, again[0]) and torch.equal(h, again[1])


def test_refusals(dev):
    x, w = torch.zeros(4, 64, dtype=F16, device=dev), torch.ones(64, dtype=F16, device=dev)
    good = dict(x=x, weight=w, block=x.clone())
    block_norm(**good)
    for kw, message in ((dict(x=x.float()), "No suitable kernel"), (dict(x=x[0]), r"\[tokens, width\]"), (dict(weight=w.double()), "No suitable kernel"),
                        (dict(weight=w[:63]), "x's width"), (dict(weight=w.cpu()), "CUDA tensor"), (dict(block=x[:3]), "x's shape"),
                        (dict(block=x.bfloat16()), "No suitable kernel"), (dict(block=x.t().contiguous().t()), "contiguous"), (dict(gate=w[:3]), "gate must be"),
                        (dict(gate=torch.zeros(3, 64, dtype=F16, device=dev)), "gate must be"), (dict(gate=w[::2].repeat(2)[::2]), "gate must be"),
                        (dict(block=None, gate=w), "without block"), (dict(block=None, residual_scale=2.0), "without block"),
                        (dict(block=None, weight=None), "neither"), (dict(bias=w, weight=None), "bias without weight"),
                        (dict(block_bias=w), "without block_weight"), (dict(weight=None, out=x.clone()), "out without weight"),
                        (dict(out=x[1:]), "x's shape"), (dict(eps=-1.0), "negative"), (dict(kind="none"), "unknown norm")):
        with pytest.raises(RuntimeError, match=message):
            block_norm(**dict(good, **kw))
    wide = torch.zeros(5, 64, dtype=F16, device=dev)
    with pytest.raises(RuntimeError, match="other rows"):
        block_norm(wide[:4], w, out=wide[1:])
    with pytest.raises(RuntimeError, match="results overlap"):
        block_norm(x, w, block=x.clone(), residual_out=wide[:4], out=wide[:4])
    with pytest.raises(RuntimeError, match="overlaps a vector"):
        block_norm(x, wide[4], block=x.clone(), out=wide[1:])
