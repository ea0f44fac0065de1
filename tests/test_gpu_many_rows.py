"""GPU: more rows than one launch has threads for (a dimension's threads are counted in 32 bits)."""
import pytest
import torch

from tests.test_gpu_cache8 import empty
from valora_amd import cache8
from valora_amd.norm import block_norm
from valora_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def alike(rows, one):
    """Whether all rows are that one (by parts: a comparison's result is as long as the rows)."""
    return all(bool((part == one).all()) for part in rows.split(1 << 24))


@pytest.mark.parametrize("T,H", [((1 << 26) + 5, 8), ((1 << 25) + 3, 520)])
def test_norms(dev, T, H):
    """Four rows a workgroup of 256 threads; and a row a workgroup of 128, as many as fit a test."""
    x, w = torch.randn(1, H, device=dev).to(BF16), torch.randn(H, device=dev).to(BF16)
    want_r, want_h = block_norm(x, w, block=x, gate=w)
    gate = w[None].expand(T, H)
    r, h = block_norm(x.expand(T, H), w, block=x.expand(T, H), gate=gate)
    assert alike(r, want_r) and alike(h, want_h)


def test_tokens_stored(dev):
    """A token a workgroup, by elements (22 of 32 are rotated)."""
    T, d = (1 << 24) + 3, 32
    one = torch.randn(3, 1, d, device=dev).to(F16)
    k, v = one[1:2].expand(T, 1, d), one[2:3].expand(T, 1, d)
    rotary = Rotary(d, rotary_dim=22, device=dev)
    loc = torch.arange(T, device=dev).flip(0)
    kc, vc, powers = empty(dev, T // 2 + 1, 1, 2, d)
    positions = torch.full((T,), 7, device=dev)
    q_out = torch.full((T, 1, d), 9.0, dtype=F16, device=dev)
    rotary.store8(positions, one[:1].expand(T, 1, d), k, v, kc, vc, powers, loc, q_out=q_out)
    want = empty(dev, 1, 1, 2, d)
    q_one = torch.empty(1, 1, d, dtype=F16, device=dev)
    rotary.store8(positions[:1], one[:1], one[1:2], one[2:3], *want, torch.zeros(1, dtype=torch.long, device=dev), q_out=q_one)
    assert alike(q_out, q_one)
    for got, its in zip((kc, vc, powers), want):
        rows = got.view(torch.uint8).view(2 * (T // 2 + 1), -1)
        assert alike(rows[:T], its.view(torch.uint8).view(2, -1)[0])
        assert alike(rows[T:], its.view(torch.uint8).view(2, -1)[1])


def test_tokens_read(dev):
    """64 tokens a workgroup of 256 threads: the results are 64 GB each."""
    n, d = (1 << 30) + 70, 32
    kc, vc, powers = empty(dev, 2, 1, 2, d)
    g = torch.Generator(device=dev).manual_seed(1)
    for codes in (kc, vc):
        codes.view(torch.uint8).copy_(torch.randint(0, 120, codes.shape, generator=g, device=dev))
    powers.view(torch.uint8).fill_(127)
    loc = torch.full((n,), 1, device=dev)
    loc[-70:] = torch.arange(70, device=dev) % 4
    k, v = cache8.read(kc, vc, powers, loc, F16)
    want = cache8.read(kc, vc, powers, torch.arange(4, device=dev), F16)
    for got, its in zip((k, v), want):
        assert torch.equal(got[-70:], its[loc[-70:]])
        for at in (0, 1 << 29, (1 << 30) - 1000):
            assert bool((got[at:at + 100] == its[1]).all())
        assert alike(got[:-70], its[1])


def test_tokens_rotated(dev):
    """q elsewhere, k and v into rows: a token a workgroup of 256 threads."""
    T, d = (1 << 24) + 3, 32
    one = torch.randn(3, 1, d, device=dev).to(F16)
    rotary = Rotary(d, device=dev)
    positions, loc = torch.full((T,), 7, device=dev), torch.arange(T, device=dev).flip(0)
    q_out, kb, vb = (torch.full((T + extra, 1, d), 9.0, dtype=F16, device=dev) for extra in (0, 1, 1))
    rotary.store(positions, one[:1].expand(T, 1, d), one[1:2].expand(T, 1, d), one[2:].expand(T, 1, d), kb, vb, loc, q_out=q_out)
    turned = one.clone()
    rotary.apply(torch.full((3,), 7, device=dev), turned)
    for rows, want in ((q_out, turned[0]), (kb, turned[1]), (vb, one[2])):
        assert alike(rows[:T], want) and alike(rows[T:], torch.full_like(want, 9.0))
