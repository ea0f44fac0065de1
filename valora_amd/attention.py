"""Attention of a batch's new tokens over the paged key/value cache.

The cache is the pool the adapters live in: a cached token is a row of ``key_buffer[layer]`` / ``value_buffer[layer]``
(``[rows, kv_heads, head_dim]``, valora/common/mem_allocator.py:243-258), and a request's rows are named by its line of a
page table.  ``AttentionPlan`` is to attention what ``LoraPlan`` is to the adapters: made once per forward pass from the lengths of
the batch, on the device, and used by every layer.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._ext import binding as _b


class AttentionPlan:
    """Cuts the attention of a batch into even pieces of work.

    Request b's new tokens are rows ``b_start_loc[b] .. + b_seq_len[b] - 1`` of q, and the last ``b_seq_len[b]`` of its
    ``b_kv_len[b]`` cached tokens (int32 device tensors, one entry per request; ``b_seq_len[b] == 0`` leaves a request out,
    so a fixed set of slots can serve a changing batch).  New token i sees the cached tokens up to itself, and with
    ``window > 0`` the last ``window`` of those only.  ``max_seq_len`` and ``max_kv_len`` bound the lengths on the host:
    grids, table and workspace go by them, the work itself by the lengths on the device.  A request with more new tokens than
    ``max_seq_len`` is left out; cached tokens beyond ``max_kv_len`` do not count.  Requests' rows must not overlap.

    Query head h reads key head ``h // (q_heads // kv_heads)``.  ``head_dim`` is 32, 64, 96, 128 or 256; ``page_size`` a power of two
    up to 256 (1: the table names pool rows, as ``MemoryAllocator.alloc`` hands them out).

    Calls that share a plan must not overlap in time (they share its workspace): one plan per stream.  The first call with
    ``weights`` takes a workspace of its own, up to 256 MB larger.
    """

    def __init__(self, b_start_loc: torch.Tensor, b_seq_len: torch.Tensor, b_kv_len: torch.Tensor, n_tokens: int, max_seq_len: int,
                 max_kv_len: int, q_heads: int, kv_heads: int, head_dim: int, page_size: int = 1, window: int = 0):
        self._native = _b.NativeAttentionPlan(b_start_loc, b_seq_len, b_kv_len, n_tokens, max_seq_len, max_kv_len, q_heads, kv_heads,
                                              head_dim, page_size, window)

    @property
    def buf(self) -> torch.Tensor:
        return self._native.buf

    @property
    def workspace(self) -> torch.Tensor:
        return self._native.workspace

    def rebuild(self) -> None:
        """Cuts the work again, in place, for what the length tensors hold now: one launch on the current stream, no
        allocation, so it can stand at the head of a captured decode step."""
        self._native.rebuild()

    def attend(self, out: torch.Tensor, q: torch.Tensor, key_buffer: torch.Tensor, value_buffer: torch.Tensor, table: torch.Tensor,
               scale: Optional[float] = None, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``out[t, h] = sum_j softmax_j(scale * q[t, h] . k_j) v_j`` over what token t sees; returns ``out``.

        ``q``, ``out`` ``[n_tokens, q_heads, head_dim]`` (or the last two flattened; rows may be apart), ``table`` int32
        ``[requests, pages]``.  ``scale`` defaults to ``head_dim ** -0.5``.  A token whose page is not in the pool is seen by
        no one; a row that sees nothing becomes zeros, as does one whose scores are all -infinity; rows of ``out`` that
        belong to no request keep their contents.  What no row sees does not show in ``out``, whatever it holds.

        ``weights`` (float32 ``[requests, >= max_kv_len]``): ``weights[b, j]`` grows by the attention that request b's rows
        give to its cached token j, summed over the heads -- what ``valora_amd.kv_cache.evict`` goes by.  A row that comes out as no
        number makes the weights of what it sees none; one whose scores lie beyond 2^22, where 32 bits do not hold the logarithm of its
        sum, adds none."""
        self._native.attend(out, q, key_buffer, value_buffer, table, scale, weights)
        return out
