"""The served requests' key/value cache, in rows of the pool that the adapters live in.

The reference keeps adapters and cached tokens in one pool of rows (``MemoryAllocator``,
valora/common/mem_allocator.py:10-27,243-258): whoever needs rows allocates them, and what is given up serves either.
``KVCache`` holds a fixed number of request slots over such a pool -- a page table whose pages are rows, the lengths, and
how much attention each cached token has got -- and makes per forward pass the ``attention`` callable that
``valora_amd.layer.layer_forward`` takes:

    cache = KVCache(mem, max_requests=64, max_len=4096, q_heads=32, rotary=Rotary(128), track=True)
    step = cache.step([0, 3], [512, 1])                # slot 0 brings a prompt, slot 3 one token
    for layer in range(n_layers):
        x = layer_forward(x, w[layer], pools[layer], plans, step.attention(layer), heads)
    cache.evict(budget=2048, recent=256, sinks=4)      # between passes
    cache.release(3)

``evict`` alone works on any paged cache whose table and weights the caller keeps.

With ``codes=True`` the cache is in 8 bits (``valora_amd.cache8``): a row holds two tokens, so the same pool holds twice as many, and passes over
it read half the bytes.
"""
from __future__ import annotations

import contextlib
from typing import Callable, ContextManager, Optional, Sequence, Tuple

import torch

from . import _lib, cache8
from ._ext import binding as _b
from .attention import AttentionPlan
from .infer_adapter import MemoryAllocator
from .rotary import Rotary


def evict(table: torch.Tensor, b_kv_len: torch.Tensor, weights: torch.Tensor, budget: int, recent: int, sinks: int = 0,
          page_size: int = 1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Requests that hold more than ``budget`` pages keep their first ``sinks`` pages, their last ``recent`` (at least one) and, of
    those between, the pages whose tokens' weights add up to most (ties: the page that comes first; what is not a number counts
    least), in their order.  One launch; nothing is moved.

    ``table`` int32 ``[requests, pages]``, ``b_kv_len`` int32 (tokens), ``weights`` float32 ``[requests, pages * page_size]``.
    Returns new tensors ``(table, b_kv_len, weights, freed)``: the pages that stay, -1 behind them; the tokens left; their
    weights, 0 behind them; the pages given up, -1 behind them."""
    return _b.cache_evict(table, b_kv_len, weights, budget, recent, sinks, page_size)


def _on(device: torch.device) -> ContextManager:
    """The pool's launches go to the current device; here it is the pool's own."""
    return torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext()


class CacheStep:
    """One forward pass over the cache: its tokens' rows and positions, and the plan of its attention.  Good until the cache's
    next ``step``, ``evict`` or ``release``."""

    def __init__(self, cache: "KVCache", positions: torch.Tensor, loc: torch.Tensor, plan: AttentionPlan):
        self.cache, self.positions, self.loc, self.plan = cache, positions, loc, plan
        self._changes = cache._changes

    def attention(self, layer: int) -> Callable[[torch.Tensor, torch.Tensor, torch.Tensor], torch.Tensor]:
        """``attend(q, k, v)`` of a layer, on the projections' outputs ``[T, heads * head_dim]`` before any rotation: rotates q and
        k, stores k and v, attends over the cache."""
        c = self.cache
        key_buffer, value_buffer, powers = c.layer(layer)

        def attend(q, k, v):
            if self._changes != c._changes:
                raise RuntimeError("the cache has changed since this step was made")
            turned, out = torch.empty_like(q), torch.empty_like(q)
            if powers is not None:
                c.rotary.store8(self.positions, q, k, v, key_buffer, value_buffer, powers, self.loc, q_out=turned)
                return self.plan.attend8(out, turned, key_buffer, value_buffer, powers, c.table, weights=c.weights)
            c.rotary.store(self.positions, q, k, v, key_buffer, value_buffer, self.loc, q_out=turned)
            return self.plan.attend(out, turned, key_buffer, value_buffer, c.table, weights=c.weights)

        return attend


class KVCache:
    """``max_requests`` slots of up to ``max_len`` cached tokens each, over the rows of ``mem`` (``head_num`` and ``head_dim`` of
    which are the key heads').  With ``track`` the attention that cached tokens get is added up over layers and passes, which
    ``evict`` goes by.  With ``codes`` tokens are kept in 8 bits, two a row, with four bytes a row and key head of every layer
    beside the pool.  Heads, types and sizes that attention does not take are refused when the cache is made.  All calls go to
    the pool's device, whichever is current, and the current stream on it; one cache serves one stream."""

    def __init__(self, mem: MemoryAllocator, max_requests: int, max_len: int, q_heads: int, rotary: Rotary, window: int = 0,
                 track: bool = False, codes: bool = False):
        if rotary.head_dim != mem.head_dim:
            raise RuntimeError(f"the rotary's head_dim={rotary.head_dim} is not the pool's {mem.head_dim}")
        if rotary.freqs.device != mem.key_buffer.device:
            raise RuntimeError(f"the rotary is on {rotary.freqs.device}, the pool on {mem.key_buffer.device}")
        if _lib.dtype_code(mem.dtype) < 0:
            raise RuntimeError(f"No suitable kernel. kv_cache: dtype={mem.dtype}")
        # heads and sizes that attention has no kernel for are refused here, not by the first step
        self.page = cache8.ROW_TOKENS if codes else 1      # tokens a row
        if not _lib.lib().mlora_attention_plan_bytes(_lib.AttentionPlan(None, 0, max_requests, 0, 0, max_len, q_heads, mem.head_num,
                                                                        mem.head_dim, self.page, window)):
            raise RuntimeError(_lib.lib().mlora_last_error().decode("utf-8", "replace"))
        self.mem, self.max_len, self.q_heads, self.rotary, self.window = mem, max_len, q_heads, rotary, window
        dev = mem.device
        pages = self._rows(max_len)
        self.table = torch.full((max_requests, pages), -1, dtype=torch.int32, device=dev)
        self.weights: Optional[torch.Tensor] = torch.zeros(max_requests, pages * self.page, device=dev) if track else None
        self.powers: Optional[torch.Tensor] = None
        if codes:
            layers, rows, heads, _ = mem.key_buffer.shape
            self.powers = cache8.new_powers((layers, rows, heads, self.page), dev)
        self.lens = [0] * max_requests           # cached tokens, and
        self.seen = [0] * max_requests           # tokens so far, evicted ones too: the next token's position
        self._changes = 0

    def _rows(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def layer(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
        """A layer's keys and values as the attention calls take them, and with ``codes`` their powers."""
        key_buffer, value_buffer = self.mem.key_buffer[layer], self.mem.value_buffer[layer]
        if self.powers is None:
            return key_buffer, value_buffer, None
        return cache8.codes_of_rows(key_buffer), cache8.codes_of_rows(value_buffer), self.powers[layer]

    def read(self, slot: int, layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(k, v)``, ``[tokens, kv_heads, head_dim]`` of the pool's type: what the slot's cached tokens hold in a layer, new tensors."""
        self._check_slot(slot)
        key_buffer, value_buffer, powers = self.layer(layer)
        n = self.lens[slot]
        rows = self.table[slot, :self._rows(n)].to(torch.long)
        if powers is None:
            return key_buffer[rows], value_buffer[rows]
        loc = (rows[:, None] * self.page + torch.arange(self.page, device=rows.device)).flatten()[:n].contiguous()
        return cache8.read(key_buffer, value_buffer, powers, loc, self.mem.dtype)

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < len(self.lens):
            raise RuntimeError(f"slot {slot} is outside [0, {len(self.lens)})")

    def step(self, slots: Sequence[int], seq_lens: Sequence[int]) -> CacheStep:
        """Rows for ``seq_lens[i]`` new tokens of slot ``slots[i]``, whose tokens follow each other in the pass's rows in this
        order.  Raises as ``MemoryAllocator.alloc`` does when the pool is full.  Whatever it raises, nothing has changed then:
        neither the pool nor the cache, and the step before is still good."""
        slots, seq_lens = [int(s) for s in slots], [int(n) for n in seq_lens]
        if len(slots) != len(seq_lens) or len(set(slots)) != len(slots):
            raise RuntimeError("step takes distinct slots with one length each")
        for s, n in zip(slots, seq_lens):
            self._check_slot(s)
            if n < 1 or self.lens[s] + n > self.max_len:
                raise RuntimeError(f"slot {s}: {n} new tokens behind {self.lens[s]}, max_len={self.max_len}")
        total = sum(seq_lens)
        lens, seen = list(self.lens), list(self.seen)
        start, new = [0] * len(lens), [0] * len(lens)
        positions, at = [], 0
        new_rows, new_columns = [], []                      # where in the table the pool's rows go
        old_rows, old_columns = [], []                      # rows of the table that have room for a token
        source, place = [], []                              # of each token: its row, among the old ones or behind them the new; where in it
        page = self.page
        n_old = sum(lens[s] % page > 0 for s in slots) if page > 1 else 0
        for s, n in zip(slots, seq_lens):
            start[s], new[s] = at, n
            first = lens[s]
            if page > 1:
                room = min(-first % page, n)                # tokens that go into the last row
                if room:
                    source += [len(old_rows)] * room
                    old_rows.append(s)
                    old_columns.append(first // page)
                fresh = n_old + len(new_rows)
                source += [fresh + i // page for i in range(n - room)]
                place += [c % page for c in range(first, first + n)]
                columns = range(self._rows(first), self._rows(first + n))
            else:
                columns = range(first, first + n)
            new_rows += [s] * len(columns)
            new_columns += columns
            positions += range(seen[s], seen[s] + n)
            at += n
            lens[s] += n
            seen[s] += n
        dev = self.mem.device
        # (one copy to the device: each costs as much as a launch or more)
        if page > 1:
            lists = [positions, new_rows, new_columns, old_rows, old_columns, source, place]
            positions, new_rows, new_columns, old_rows, old_columns, source, place = \
                torch.tensor(sum(lists, []), dtype=torch.long).to(dev).split([len(l) for l in lists])
        else:
            positions, new_rows, new_columns = torch.tensor([positions, new_rows, new_columns], dtype=torch.long).to(dev)
        lengths = torch.tensor([start, new, lens], dtype=torch.int32).to(dev)
        plan = AttentionPlan(lengths[0], lengths[1], lengths[2], n_tokens=total, max_seq_len=max(seq_lens, default=0),
                             max_kv_len=max((lens[s] for s in slots), default=0), q_heads=self.q_heads,
                             kv_heads=self.mem.head_num, head_dim=self.mem.head_dim, page_size=self.page, window=self.window)
        with _on(dev):
            got = self.mem.alloc(new_rows.numel())
            try:
                loc = got
                if page > 1:
                    loc = torch.cat([self.table[old_rows, old_columns].to(torch.long), got])[source] * page + place
                self.table[new_rows, new_columns] = got.to(torch.int32)
            except BaseException:
                self.mem.free(got)
                raise
        self.lens, self.seen = lens, seen
        self._changes += 1
        return CacheStep(self, positions, loc, plan)

    def evict(self, budget: int, recent: int, sinks: int = 0) -> int:
        """Every slot with more than ``budget`` cached tokens gives up those that got the least attention (see the function
        ``evict``); their rows go back to the pool.  Returns how many rows.  With ``codes`` it goes by rows of two tokens: the budget is rounded
        down to them, ``recent`` and ``sinks`` up.  Positions go on from where they were.  Nothing has changed where it raises."""
        if self.weights is None:
            raise RuntimeError("evict needs a cache that was made with track=True")
        if self.window > 0:
            raise RuntimeError("evict and window exclude each other: a window counts cached tokens")
        lens = torch.tensor(self.lens, dtype=torch.int32).to(self.mem.device)
        if self.page > 1:
            budget //= self.page
            recent, sinks = (self._rows(n) if n > 0 else n for n in (recent, sinks))      # (negative ones are refused below)
        table, _, weights, freed = evict(self.table, lens, self.weights, budget, recent, sinks, self.page)
        over = [max(0, self._rows(n) - budget) for n in self.lens]
        count = sum(over)
        if count:
            self._free(freed.view(-1), count)
        self.table, self.weights = table, weights
        self.lens = [n - k * self.page for n, k in zip(self.lens, over)]
        self._changes += 1
        return count

    def release(self, slot: int) -> None:
        """The slot's rows go back to the pool; the slot is empty."""
        self._check_slot(slot)
        n = self._rows(self.lens[slot])
        if n:
            self._free(self.table[slot, :n], n)
            self.table[slot] = -1
            if self.weights is not None:
                self.weights[slot] = 0
        self.lens[slot] = self.seen[slot] = 0
        self._changes += 1

    def _free(self, rows: torch.Tensor, count: int) -> None:
        """``count`` rows among ``rows`` (others are -1, which the pool leaves out)."""
        mem, rows = self.mem, rows.to(torch.long)
        with _on(mem.device):
            _lib.check(_lib.lib().mlora_pool_free(_lib.current_stream(mem.device), _lib.ptr(mem.mem_state), mem.tot_size, _lib.ptr(rows),
                                                  rows.numel()))
        mem.can_use_mem_size += count
