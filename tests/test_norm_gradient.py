"""The norms have no backward pass: where a gradient would be recorded they refuse, before anything else is looked at, instead of dropping it."""
import pytest
import torch

from valora_amd.layer import LayerWeights, layer_forward
from valora_amd.norm import block_norm


@pytest.mark.parametrize("name", ["x", "weight", "bias", "block", "block_weight", "block_bias", "gate", "residual_out", "out"])
def test_an_operand_that_requires_a_gradient(name):
    rows, vectors = ("x", "block", "residual_out", "out"), ("weight", "bias", "block_weight", "block_bias", "gate")
    t = {n: torch.zeros(2, 8, dtype=torch.float16) for n in rows}
    t.update({n: torch.zeros(8, dtype=torch.float16) for n in vectors})
    t[name].requires_grad_()
    with pytest.raises(RuntimeError, match=f"no backward pass: {name} requires"):
        block_norm(**t)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
        block_norm(**t)


def test_a_fused_layer():
    """Which without ``fused`` carries the gradient."""
    z = torch.eye(4, dtype=torch.float64)
    w = LayerWeights(z, z, z, z, z, z, z, z[0], z[0])
    x = torch.ones(4, 4, dtype=torch.float64, requires_grad=True)
    layer_forward(x, w, None, None, lambda q, k, v: q, 1).sum().backward()
    assert x.grad is not None
    with pytest.raises(RuntimeError, match="no backward pass"):
        layer_forward(x, w, None, None, lambda q, k, v: q, 1, fused=True)
