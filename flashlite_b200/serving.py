"""A paged key/value cache and the serving step over it.

``PagedCache`` keeps what the serving operators share from step to step: the
caches of every layer, the block table, the free list and the requests'
lengths, all on the device. One step is::

    step = cache.plan(cu_seqlens, total_tokens)             # or parents=..., for trees
    for layer in range(cache.layers):
        out = cache.attend(layer, q, k, v, table, step)     # q, k, v of the new tokens
    cache.commit(step, kept)                                # how many each request keeps

None of these waits for the GPU, and the state is updated where it lies, so that
a step captured into a CUDA graph goes on from replay to replay (``release``
waits, and is called between replays). With drafted trees, ``commit`` also takes
the kept path of each request, whose keys and values move next to the cached
ones. No reference counterpart: the reference has no cache.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .flash_attn_wmma import plan_cache_step, rotary_append, settle_step, tree_attention


class Step(NamedTuple):
    """What ``PagedCache.plan`` found for the new tokens of one step."""

    cu_seqlens: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    admitted: torch.Tensor
    tree_mask: torch.Tensor | None
    context_lens: torch.Tensor | None = None  # cached tokens, -1 for a refused request: as attention takes them


class PagedCache:
    """Keys and values of up to ``requests`` requests in ``num_blocks`` blocks of ``page_size`` tokens per layer.

    ``layout`` "bnhd" stores a block as ``[page, heads, D]``, "bhnd" as
    ``[heads, page, D]``.
    """

    def __init__(self, requests: int, num_blocks: int, page_size: int, kv_heads: int, head_dim: int,
                 max_blocks: int, layers: int = 1, dtype: torch.dtype = torch.float16, layout: str = "bnhd",
                 device="cuda"):
        if layout not in ("bhnd", "bnhd"):
            raise ValueError("layout must be 'bhnd' or 'bnhd'")
        shape = (page_size, kv_heads) if layout == "bnhd" else (kv_heads, page_size)
        self.layers, self.page_size, self.layout = layers, page_size, layout
        # one block more than is given out: copies that are none land there (commit)
        self.spare = num_blocks * page_size
        with torch.inference_mode(False):  # a cache made in that mode can be written outside of it
            self.k = [torch.zeros((num_blocks + 1, *shape, head_dim), dtype=dtype, device=device) for _ in range(layers)]
            self.v = [torch.zeros_like(k) for k in self.k]
            ints = dict(dtype=torch.int32, device=device)
            self.block_table = torch.zeros((requests, max_blocks), **ints)
            self.context_lens = torch.zeros(requests, **ints)
            self.held_blocks = torch.zeros(requests, **ints)
            self.free_blocks = torch.arange(num_blocks - 1, -1, -1, **ints)
            self.num_free = torch.full((1,), num_blocks, **ints)

    def plan(self, cu_seqlens: torch.Tensor, total_tokens: int, parents: torch.Tensor | None = None,
             mask_words: int = 0) -> Step:
        """Blocks, slots and positions for the new tokens ``cu_seqlens[b]:cu_seqlens[b+1]`` of each request."""
        slots, positions, admitted, num_free, held_blocks, mask = plan_cache_step(
            self.context_lens, cu_seqlens, self.block_table, self.held_blocks, self.free_blocks, self.num_free,
            total_tokens, self.page_size, parents=parents, mask_words=mask_words)
        lens = settle_step(self.context_lens, self.held_blocks, self.num_free, admitted, held_blocks, num_free)
        return Step(cu_seqlens, slots, positions, admitted, mask, lens)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, step: Step,
               interleaved: bool = False, sm_scale: float = 0.0) -> torch.Tensor:
        """Rotates ``q`` and ``k``, appends ``k`` and ``v`` to the layer's cache and attends to it. The rows of a refused
        request are 0."""
        lens = self.context_lens if step.context_lens is None else step.context_lens
        q = rotary_append(q, k, v, table, step.positions, step.slots, self.k[layer], self.v[layer],
                          interleaved=interleaved, layout=self.layout)
        out, _ = tree_attention(q, self.k[layer], self.v[layer], self.block_table, lens, step.cu_seqlens,
                                tree_mask=step.tree_mask, sm_scale=sm_scale, layout=self.layout)
        return out

    def commit(self, step: Step, kept: torch.Tensor, path: torch.Tensor | None = None) -> None:
        """Request b keeps its first ``kept[b]`` new tokens, or, with ``path`` ``[requests, n]``, the new tokens
        ``path[b, :kept[b]]`` (indices within the request, from the root down). A refused request keeps none.
        """
        kept = torch.where(step.admitted, kept, 0).to(torch.int32)
        if path is not None and step.slots.numel() > 0:
            first = step.cu_seqlens[:-1, None].long()
            column = torch.arange(path.shape[1], device=path.device)
            live = column < kept[:, None]
            last = step.slots.numel() - 1
            source = step.slots[torch.where(live, first + path, 0).clamp(0, last)]
            target = step.slots[torch.where(live, first + column, 0).clamp(0, last)]
            # entries past a request's path copy the spare block's first row onto itself
            source, target = (torch.where(live, s, self.spare) for s in (source, target))
            sb, sr, tb, tr = source // self.page_size, source % self.page_size, target // self.page_size, \
                target % self.page_size
            for cache in (*self.k, *self.v):
                if self.layout == "bnhd":
                    cache[tb, tr] = cache[sb, sr]
                else:
                    cache[tb, :, tr] = cache[sb, :, sr]
        self.context_lens += kept

    def release(self, request: int) -> None:
        """Gives a finished request's blocks back. Reads its length, so it waits for the GPU."""
        held, free = int(self.held_blocks[request]), int(self.num_free)
        self.free_blocks[free:free + held] = self.block_table[request, :held]
        self.num_free += held
        self.context_lens[request] = 0
        self.held_blocks[request] = 0
