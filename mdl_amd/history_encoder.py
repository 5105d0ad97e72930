"""A history encoder on the operators of this package.

``ShardedEmbedding`` rows of a user's events, then blocks of gated window
attention between fused norms:

    h, mask = encoder(ids, lengths)                 # training, or a prompt
    caches = encoder.caches(batch)                  # serving:
    h = encoder.prefill(ids, lengths, caches)       #   histories so far, at once
    h = encoder.step(new_ids, positions, caches)    #   then one event a user

``step`` answers an event as the whole history's ``encoder`` would (to the
rounding of the dtype): position ``p`` of a history stands in column ``p`` of
its right-aligned window, less the padding.  The event table trains with
``ShardedRowWiseAdagrad`` (its gradient is sparse), the other parameters with
any optimizer.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor, nn

from .block_norm import gated_residual_norm
from .embeddings import ShardedEmbedding, sequence_embedding_lookup
from .history import HistoryCache, RelativeBuckets, history_attention


class HistoryBlock(nn.Module):
    """Attention from a normalised input, and the norms and gate after it.

    ``forward(x, h, mask)`` takes the residual stream ``x [B, T, dim]`` and its
    norm ``h`` and returns both for the next block.
    """

    def __init__(self, dim: int, heads: int, *, kv_heads: Optional[int] = None, head_dim: Optional[int] = None,
                 window: Optional[int] = None, sinks: int = 0, buckets: Optional[RelativeBuckets] = None,
                 dtype: Optional[torch.dtype] = None) -> None:
        super().__init__()
        self.heads = heads
        self.kv_heads = heads if kv_heads is None else kv_heads
        self.head_dim = dim // heads if head_dim is None else head_dim
        self.window = window
        self.sinks = sinks
        self.buckets = buckets
        inner = self.heads * self.head_dim
        self.qkv = nn.Linear(dim, inner + 2 * self.kv_heads * self.head_dim, bias=False, dtype=dtype)
        self.gate = nn.Linear(dim, dim, dtype=dtype)
        self.out = nn.Linear(inner, dim, bias=False, dtype=dtype)
        self.post_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        self.next_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        self.residual_scale = nn.Parameter(torch.full((dim,), 0.5, dtype=dtype))
        self.bias_table = None
        if buckets is not None:
            self.bias_table = nn.Parameter(torch.zeros(buckets.num_buckets, heads, dtype=dtype))

    def _heads(self, h: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        # views of one product: the operators take rows and heads at any stride
        sizes = (self.heads, self.kv_heads, self.kv_heads)
        return self.qkv(h).unflatten(-1, (sum(sizes), self.head_dim)).split(sizes, -2)

    def _after(self, x: Tensor, h: Tensor, attended: Tensor) -> tuple[Tensor, Tensor]:
        return gated_residual_norm(x, self.out(attended.flatten(-2)), self.post_weight, self.next_weight,
                                   gate=self.gate(h), residual_scale=self.residual_scale)

    def forward(self, x: Tensor, h: Tensor, mask: Tensor) -> tuple[Tensor, Tensor]:
        q, k, v = self._heads(h)
        attended = history_attention(q, k, v, mask=mask, window=self.window, sinks=self.sinks,
                                     bias_table=self.bias_table, buckets=self.buckets)
        return self._after(x, h, attended)

    def prefill(self, x: Tensor, h: Tensor, mask: Tensor, lengths: Tensor, cache: HistoryCache
                ) -> tuple[Tensor, Tensor]:
        q, k, v = self._heads(h)
        cache.write(k, v, lengths, right_aligned=True)
        attended = history_attention(q, k, v, mask=mask, window=self.window, sinks=self.sinks,
                                     bias_table=self.bias_table, buckets=self.buckets)
        return self._after(x, h, attended)

    def step(self, x: Tensor, h: Tensor, positions: Tensor, cache: HistoryCache) -> tuple[Tensor, Tensor]:
        q, k, v = self._heads(h)
        attended = cache.step(q, k, v, positions, bias_table=self.bias_table, buckets=self.buckets)
        return self._after(x, h, attended)


class HistoryEncoder(nn.Module):
    """Event embeddings and ``depth`` blocks (see the module docstring)."""

    def __init__(self, events: ShardedEmbedding, depth: int, heads: int, **block) -> None:
        super().__init__()
        self.events = events
        dim, dtype = events.embedding_dim, events.weight.dtype
        self.first_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        self.blocks = nn.ModuleList(HistoryBlock(dim, heads, dtype=dtype, **block) for _ in range(depth))

    def _embed(self, ids: Tensor, lengths: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        x, mask = sequence_embedding_lookup(self.events, ids, lengths)
        x, h = gated_residual_norm(x, None, None, self.first_weight)
        return x, h, mask

    def forward(self, ids: Tensor, lengths: Tensor) -> tuple[Tensor, Tensor]:
        """``([B, T, dim], [B, T] mask)`` of right-padded ids, right-aligned."""

        x, h, mask = self._embed(ids, lengths)
        for block in self.blocks:
            x, h = block(x, h, mask)
        return h, mask

    def caches(self, batch: int, capacity: Optional[int] = None) -> list[HistoryCache]:
        """One cache a block; without ``capacity`` just what a window sees."""

        made = []
        for block in self.blocks:
            slots = capacity
            if slots is None:
                if block.window is None:
                    raise ValueError("blocks without a window need a cache capacity")
                slots = block.sinks + block.window
            made.append(HistoryCache.empty(batch, slots, block.kv_heads, block.head_dim, window=block.window,
                                           sinks=block.sinks, dtype=self.first_weight.dtype,
                                           device=self.first_weight.device))
        return made

    @torch.no_grad()
    def prefill(self, ids: Tensor, lengths: Tensor, caches: Sequence[HistoryCache]) -> Tensor:
        x, h, mask = self._embed(ids, lengths)
        for block, cache in zip(self.blocks, caches):
            x, h = block.prefill(x, h, mask, lengths, cache)
        return h

    @torch.no_grad()
    def step(self, ids: Tensor, positions: Tensor, caches: Sequence[HistoryCache]) -> Tensor:
        """``[B, dim]`` of one new event a user, at ``positions [B]``."""

        x, h = gated_residual_norm(self.events(ids), None, None, self.first_weight)
        for block, cache in zip(self.blocks, caches):
            x, h = block.step(x, h, positions, cache)
        return h
