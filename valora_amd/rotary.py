"""Rotary positions, written straight into the paged cache.

A served layer rotates q and k of its new tokens by their positions and keeps the rotated k and the v as rows of the pool
(``MemoryAllocator.key_buffer[layer]`` / ``value_buffer[layer]``, valora/common/mem_allocator.py:243-258).  ``Rotary.store``
does both in one launch: q is rotated in place (or into ``q_out``), k and v go from the projections' output to the tokens'
rows without a copy in between.  ``Rotary.apply`` is the rotation alone.

Angles are exact at any position: position times frequency is reduced to a fraction of a turn in 64 bits on the device.
"""
from __future__ import annotations

import math
from typing import Dict, Optional

import torch

from ._ext import binding as _b


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Dict] = None):
    """``(radians per position of each pair, gain of sine and cosine)``.

    ``base ** (-2 i / rotary_dim)`` for pair i, and with ``scaling`` what stretches it over a longer context
    (``factor`` = new length / trained length):

    * ``{"type": "linear", "factor"}``: every frequency divided by the factor
    * ``{"type": "ntk", "factor"}``: the base times ``factor ** (rotary_dim / (rotary_dim - 2))``, so that the lowest frequency
      is divided by the factor and the highest kept
    * ``{"type": "bands", "factor", "low", "high", "original_max_position"}``: pairs that turn more than ``high`` times in the
      original context are kept, those that turn less than ``low`` times divided by the factor, those between interpolated
      by their turns
    * ``{"type": "yarn", "factor", "original_max_position", "beta_fast" = 32, "beta_slow" = 1, "attention_factor" = None}``:
      kept below the dimension that turns ``beta_fast`` times, divided from the one that turns ``beta_slow`` times on,
      interpolated by dimension between; gain ``0.1 ln(factor) + 1``, 1 for factors below 1, unless
      ``attention_factor`` gives it
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim={rotary_dim} must be even and positive")
    if not base > 0:
        raise RuntimeError(f"base={base} must be positive")
    plain = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return plain, 1.0
    s = dict(scaling)
    kind, factor = s.pop("type", None), float(s.pop("factor", 0.0))
    if kind not in ("linear", "ntk", "bands", "yarn"):
        raise RuntimeError(f"unknown rotary scaling {kind!r}")
    if not (factor > 0 and math.isfinite(factor)):
        raise RuntimeError(f"rotary scaling needs a positive factor, got {factor}")
    gain = 1.0
    if kind == "linear":
        out = [f / factor for f in plain]
    elif kind == "ntk":
        if rotary_dim < 4:
            raise RuntimeError("ntk scaling needs more than one pair")
        stretched = base * factor ** (rotary_dim / (rotary_dim - 2.0))
        out = [stretched ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    else:
        try:
            context = float(s.pop("original_max_position"))
        except KeyError:
            raise RuntimeError(f"{kind} scaling needs original_max_position") from None
        if not context > 0:
            raise RuntimeError(f"{kind} scaling needs a positive original_max_position, got {context}")
        if kind == "bands":
            low, high = float(s.pop("low", 1.0)), float(s.pop("high", 4.0))
            if not high > low:
                raise RuntimeError("bands scaling needs high > low")
            share = [min(1.0, max(0.0, (context * f / (2 * math.pi) - low) / (high - low))) for f in plain]   # kept
        else:
            fast, slow, given = float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0)), s.pop("attention_factor", None)
            if not (base > 1 and fast >= slow > 0):
                raise RuntimeError("yarn scaling needs base > 1 and beta_fast >= beta_slow > 0")

            def dimension(turns):
                return rotary_dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo, hi = max(math.floor(dimension(fast)), 0), min(math.ceil(dimension(slow)), rotary_dim - 1)
            share = [1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rotary_dim // 2)]
            gain = 0.1 * math.log(max(factor, 1.0)) + 1.0 if given is None else float(given)
        out = [f * t + f / factor * (1.0 - t) for f, t in zip(plain, share)]
    if s:
        raise RuntimeError(f"rotary scaling {kind}: unknown entries {sorted(s)}")
    return out, gain


class Rotary:
    """The first ``rotary_dim`` (default: all) elements of a head are rotated, in pairs ``(i, i + rotary_dim / 2)`` or, with
    ``interleaved``, ``(2 i, 2 i + 1)``; the others pass through.  ``scaling``: see ``frequencies``."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[Dict] = None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim > head_dim:
            raise RuntimeError(f"rotary_dim={rotary_dim} is more than head_dim={head_dim}")
        radians, self.gain = frequencies(rotary_dim, base, scaling)
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        self.freqs = torch.tensor(radians, dtype=torch.float64).div_(2 * math.pi).to(device)    # turns per position
        self._native = _b.NativeRotary(self.freqs, head_dim, self.interleaved, self.gain)

    def apply(self, positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> None:
        """``q`` (and ``k``) ``[T, heads, head_dim]`` or ``[T, heads * head_dim]``, any token and head strides, rotated in place
        or into ``q_out`` / ``k_out``; ``positions`` int64 ``[T]``."""
        self._native.apply(positions, q, k, q_out, k_out)

    def store(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_buffer: torch.Tensor,
              value_buffer: torch.Tensor, loc: torch.Tensor, q_out: Optional[torch.Tensor] = None) -> None:
        """Rotates q in place or into ``q_out``, and writes the rotated k and the v of token t to row ``loc[t]`` of the
        layer's ``key_buffer`` / ``value_buffer`` ``[rows, kv_heads, head_dim]``; k and v themselves stay as they are.  ``loc``
        (int64, as ``MemoryAllocator.alloc`` returns it) names each row at most once; a token whose row is outside the
        buffers is not stored."""
        self._native.store(positions, q, k, v, key_buffer, value_buffer, loc, q_out)
