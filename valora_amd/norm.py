"""The norms around a layer's blocks, in one launch with the sum they stand at.

A decoder layer adds each block's output to its residual stream and normalises the sum for the next block
(valora/models/llama/layer_infer/transformer_layer_infer.py:36-37 and its template's forward); some models normalise the block's output too,
scale it by a learned gate, or scale either side.  ``block_norm`` does all of it with each row read and written once:

    r = residual_scale * x + block_scale * gate * N(block; block_weight, block_bias)
    h = N(r; weight, bias)

    N(z; w, b) = z / sqrt(mean(z^2) + eps) * (offset + w) + b         kind="rms"
    the same of z - mean(z)                                           kind="layer"
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import binding as _b


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               block: Optional[torch.Tensor] = None, block_weight: Optional[torch.Tensor] = None, block_bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0, eps: float = 1e-6,
               kind: str = "rms", offset: float = 0.0, residual_out: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(r, h)``.  ``x``, ``block`` ``[tokens, width]``, float16 or bfloat16, rows may be apart; vectors ``[width]`` and the gate (``[width]``,
    ``[tokens, 1]`` or ``[tokens, width]``) are of that type or float32.  Without ``block`` r is ``x`` itself; without ``block_weight`` the block
    joins as it is; without ``weight`` h is None.  Everything is in 32 bits; r and h are rounded once each, h from the unrounded r.  Widths go up
    to 32768.  ``residual_out`` and ``out`` may be ``x`` or ``block`` themselves, or other columns of one tensor; results that overlap anything
    else that the call reads, or each other, are refused.  There is no backward pass: operands that require a gradient are refused where one
    would be recorded."""
    if kind not in ("rms", "layer"):
        raise RuntimeError(f"unknown norm {kind!r} (rms or layer)")
    return _b.block_norm(x, weight, bias, block, block_weight, block_bias, gate, residual_scale, block_scale, eps, kind == "layer", offset,
                         residual_out, out)
