"""Keeping sequences inside a cache budget.

A long-running sequence fills its cache with tokens of which attention uses
few.  ``CacheRecord`` stands beside one layer's paged cache and holds what is
needed to cut it: for every cached entry the attention weight it has received
(fp32) and the position it came from (int32), both [num_blocks, kv heads,
block_size].  Set as ``TurboQuantFusedImpl.record`` it is filled by ``forward``
itself:

* a prompt (or any batch with more than one query per request) through
  ``ops.track_window``: the last ``window`` queries of each chunk;
* a decode step through ``ops.decode_paged_tracked``, which returns the
  attention output too.

``evict`` then cuts every sequence that is over ``budget``: kept are the first
``sink`` positions, the last ``recent`` ones and, of the rest, the entries with
the largest weights, per kv head (``ops.evict_paged``).  The caller goes on
with the lengths that it returns; pages behind them are free.  Positions go
on counting: after a cut a sequence's next token has the position of its
tokens seen, not its cached length, so the caller passes both
(``attn_metadata.tokens_seen``, or seq_lens where nothing has been evicted).
Nothing here has a counterpart in the reference, whose cache only grows.
"""
from __future__ import annotations

import torch

from . import ops
from .geometry import BALANCED_MAX_BATCH

STARTS_KEPT = 64  # row widths whose starts a record keeps (4 KB each)


class CacheRecord:
    """Weights and positions of one layer's cache, and the rule of its cuts."""

    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, budget: int,
                 recent: int = 0, sink: int = 0, window: int = 32,
                 device: torch.device | str = "cuda:0"):
        if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
            raise ValueError(f"budget {budget} must hold recent {recent} + sink {sink} tokens")
        if window < 1:
            raise ValueError(f"window {window} must be positive")
        shape = (num_blocks, num_kv_heads, block_size)
        self.weights = torch.zeros(shape, dtype=torch.float32, device=device)
        self.positions = torch.zeros(shape, dtype=torch.int32, device=device)
        self.budget, self.recent, self.sink, self.window = budget, recent, sink, window
        self._starts: dict[int, torch.Tensor] = {}  # by row width
        self._last = None  # ((rows, width), indptr) of the last call

    @classmethod
    def beside(cls, kv_cache: torch.Tensor, budget: int, **rule) -> "CacheRecord":
        """The record of a cache [2, num_blocks, block_size, H, ebs]."""
        _, nb, bs, h, _ = kv_cache.shape
        return cls(nb, bs, h, budget, device=kv_cache.device, **rule)

    def _tables(self, block_table: torch.Tensor):
        """(indices, indptr) of a strided page table."""
        if block_table.dtype != torch.int32 or not block_table.is_contiguous():
            block_table = block_table.to(torch.int32).contiguous()
        b, width = key = tuple(block_table.shape)
        if self._last is None or self._last[0] != key:
            starts = self._starts_of(width, b, block_table)
            if starts is None:  # this call's own, on its stream
                return block_table.reshape(-1), torch.arange(
                    b + 1, dtype=torch.int32, device=block_table.device) * width
            self._last = key, starts[:b + 1]
        return block_table.reshape(-1), self._last[1]

    def _starts_of(self, width: int, rows: int, block_table: torch.Tensor):
        """Starts of up to BALANCED_MAX_BATCH rows of `width` pages, or None.  Made
        on the host and copied before the call returns, so that any stream may use
        them, but not inside a capture (a graph's memory is its own); kept for good,
        as a graph may hold them, for at most STARTS_KEPT widths."""
        if rows > BALANCED_MAX_BATCH:
            return None
        starts = self._starts.get(width)
        if starts is None and len(self._starts) < STARTS_KEPT and not (
                block_table.is_cuda and torch.cuda.is_current_stream_capturing()):
            starts = torch.arange(BALANCED_MAX_BATCH + 1, dtype=torch.int32) * width
            starts = self._starts[width] = starts.to(block_table.device)
        return starts

    def decode(self, q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor,
               seq_lens: torch.Tensor, tokens_seen: torch.Tensor, num_kv_heads: int,
               head_dim: int, padded_dim: int, sm_scale: float, signs: torch.Tensor | None,
               o: torch.Tensor) -> torch.Tensor:
        """Attention of one new token per sequence, q and o [B, Hq, head_dim]."""
        for a in range(0, q.size(0), BALANCED_MAX_BATCH):
            z = min(a + BALANCED_MAX_BATCH, q.size(0))
            indices, indptr = self._tables(block_table[a:z])
            ops.decode_paged_tracked(q[a:z], kv_cache, indices, indptr, seq_lens[a:z],
                                     num_kv_heads, head_dim, padded_dim, sm_scale, signs, o[a:z],
                                     self.weights, self.positions, tokens_seen[a:z])
        return o

    def observe(self, q: torch.Tensor, query_start_loc: torch.Tensor, kv_cache: torch.Tensor,
                block_table: torch.Tensor, seq_lens: torch.Tensor, tokens_seen: torch.Tensor,
                num_kv_heads: int, head_dim: int, padded_dim: int, sm_scale: float,
                signs: torch.Tensor | None) -> None:
        """The record of a batch of chunks, q [tokens, Hq, head_dim]."""
        most = 1024 * num_kv_heads // q.size(1)  # observed queries a call takes
        batch = query_start_loc.numel() - 1
        for a in range(0, batch, BALANCED_MAX_BATCH):
            z = min(a + BALANCED_MAX_BATCH, batch)
            indices, indptr = self._tables(block_table[a:z])
            ops.track_window(q, query_start_loc[a:z + 1], min(self.window, most), kv_cache,
                             indices, indptr, seq_lens[a:z], num_kv_heads, head_dim, padded_dim,
                             sm_scale, signs, self.weights, self.positions, tokens_seen[a:z])

    def evict(self, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
              tokens_seen: torch.Tensor, new_lens: torch.Tensor | None = None) -> torch.Tensor:
        """Cuts the sequences to the budget; returns their lengths (int32 [B],
        written into new_lens, which may be seq_lens)."""
        indices, indptr = self._tables(block_table)
        if new_lens is None:
            new_lens = torch.empty_like(seq_lens)
        return ops.evict_paged(kv_cache, self.weights, self.positions, indices, indptr, seq_lens,
                               tokens_seen, self.budget, self.recent, self.sink, new_lens)
