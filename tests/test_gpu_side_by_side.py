"""GPU: operands that are parts of one tensor, and do not overlap, are taken as separate ones are."""
import pytest
import torch

from tests.test_gpu_cache8 import empty
from valora_amd import cache8
from valora_amd.norm import block_norm
from valora_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("T", [1, 77, 5000])
def test_q_in_place_beside_k_and_v(dev, by_head, T):
    """A projection's output, q then k then v, or the three of each head; and k and v read back into the halves of one tensor."""
    heads, d, page = 4, 64, 2
    g = torch.Generator(device=dev).manual_seed(T)
    qkv = torch.randn(T, 3 * heads, d, generator=g, device=dev).to(BF16)
    q, k, v = (qkv[:, i::3] if by_head else qkv[:, i * heads:(i + 1) * heads] for i in range(3))
    positions, loc = torch.arange(T, device=dev), torch.randperm(T + 1, generator=g, device=dev)[:T]
    rotary = Rotary(d, device=dev)
    want, got = empty(dev, T // 2 + 1, heads, page, d), empty(dev, T // 2 + 1, heads, page, d)
    apart = [x.contiguous() for x in (q, k, v)]
    rotary.store8(positions, *apart, *want, loc)
    rotary.store8(positions, q, k, v, *got, loc)
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(v, apart[2])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    both = torch.full((T, 2, heads, d), 7.0, dtype=BF16, device=dev)
    cache8.read(*got, loc, BF16, both[:, 0], both[:, 1])
    rk, rv = cache8.read(*got, loc, BF16)
    assert torch.equal(both[:, 0], rk) and torch.equal(both[:, 1], rv)


@pytest.mark.parametrize("gate_width", [1, 520])
@pytest.mark.parametrize("T,H", [(1, 520), (33, 520), (40, 96)])
def test_norm_of_columns(dev, T, H, gate_width):
    """A block's output, a gate and both results in columns of one tensor.  (Where rows are no whole accesses it is another kernel, whose result may be
    the neighbour in 16 bits: a step, 2^-10 of the value, 2^-24 at least.)"""
    near = lambda a, b: bool(((a.double() - b.double()).abs() <= b.double().abs() * 2.0 ** -10 + 2.0 ** -24).all())  # noqa: E731
    gate_width = min(gate_width, H)
    g = torch.Generator(device=dev).manual_seed(T)
    wide = torch.randn(T, 4 * H + gate_width, generator=g, device=dev).to(F16)
    x, block, r, h, gate = wide.split([H, H, H, H, gate_width], 1)
    w = torch.randn(H, generator=g, device=dev).to(F16)
    want_r, want_h = block_norm(x.clone(), w, block=block.clone(), block_weight=w, gate=gate.clone())
    keep = wide.clone()
    block_norm(x, w, block=block, block_weight=w, gate=gate, residual_out=r, out=h)
    assert near(r, want_r) and near(h, want_h)
    keep[:, 2 * H:4 * H] = wide[:, 2 * H:4 * H]
    assert torch.equal(wide, keep)
    block_norm(x, w, block=block, block_weight=w, gate=gate, residual_out=x, out=block)
    assert torch.equal(x, r) and torch.equal(block, h)
