"""The key/value cache in 8 bits.

A token's k or v of a key head is held as ``head_dim`` e4m3 codes times one power of two: the least with which the head's largest finite
element is at most 448, e4m3's largest value, and within bounds that make every code times its power a value of the model's type (2^-15 to
2^7 for float16, 2^-117 to 2^119 for bfloat16).  An element is off by half a step of e4m3, 2^-4 of itself, or by 2^-10 of the power where it
is below 2^-6 of it; infinities become the largest value, what is no number stays none.

* codes   float8_e4m3fn ``[pages, kv_heads, page_size, head_dim]``, of keys and of values
* powers  float8_e8m0fnu ``[pages, kv_heads, page_size, 2]``: the keys', the values'

``valora_amd.rotary.Rotary.store8`` writes them, ``valora_amd.attention.AttentionPlan.attend8`` attends over them and ``read`` gives back the
values.  A slot is a token's place: page times page size plus the place in the page.  A pool row of 16-bit elements
(``MemoryAllocator.key_buffer``, valora/common/mem_allocator.py:243-258) holds the codes of two tokens: ``codes_of_rows`` is that view, which
``valora_amd.kv_cache.KVCache`` with ``codes=True`` keeps its tokens in.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from ._ext import binding as _b

ROW_TOKENS = 2      # tokens that a row of 16-bit elements holds the codes of


def codes_of_rows(buffer: torch.Tensor) -> torch.Tensor:
    """A pool's 16-bit rows ``[rows, kv_heads, head_dim]`` as pages of two tokens' codes, the same memory."""
    if buffer.dim() != 3 or buffer.element_size() != 2 or not buffer[:1].is_contiguous():
        raise RuntimeError("codes_of_rows takes 16-bit rows [rows, kv_heads, head_dim], each contiguous")
    rows, heads, dim = buffer.shape
    return buffer.view(torch.float8_e4m3fn).unflatten(2, (ROW_TOKENS, dim))


def new_powers(shape: Sequence[int], device) -> torch.Tensor:
    """Powers ``[..., 2]`` beside codes of the shape ``[..., kv_heads, page_size]``, all 1."""
    return torch.full((*shape, 2), 127, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)


def read(key_codes: torch.Tensor, value_codes: torch.Tensor, powers: torch.Tensor, loc: torch.Tensor, dtype: torch.dtype,
         k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, ``[n, kv_heads, head_dim]`` of ``dtype``: what the slots ``loc`` (int64 ``[n]``) hold; zeros for one outside the cache.
    Exact in the type that the cache was written from; as another type values are rounded to the nearest, beyond its largest to infinities.
    ``k_out`` and ``v_out`` may lie side by side in one tensor; they must not overlap each other, ``loc`` or the cache's pages, read or not."""
    return _b.cache8_read(key_codes, value_codes, powers, loc, dtype, k_out, v_out)
