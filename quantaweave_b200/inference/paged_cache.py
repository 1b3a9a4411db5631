"""The storage of a block-wise 8-bit KV cache and its bookkeeping for a fixed number of requests.

Per layer two code tensors ``[blocks, kv_heads, block, head_dim]`` and two scale tensors ``[blocks, kv_heads]``; one block
table, free list and plan state for all layers (a token has the same slot in each). Everything lives on the device: a step
allocates its own blocks, so it can be captured in a CUDA graph and replayed while requests grow. See ``ops.kv_cache``.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from ..ops import kv_cache as ops


class PoolExhausted(RuntimeError):
    """The pool has fewer blocks than the requests need."""


class PagedKVCache:
    """``blocks`` defaults to what ``requests`` full contexts need; with fewer, who admits requests keeps count
    (``blocks_for``) or asks before a step (``require``): a token without a block is not stored."""

    def __init__(self, layers: int, requests: int, capacity: int, kv_heads: int, head_dim: int, device,
                 fmt: str = "fp8", block: int = 64, blocks: Optional[int] = None) -> None:
        if fmt not in ops.FORMATS:
            raise ValueError(f"the cache format is one of {sorted(ops.FORMATS)}, got {fmt!r}")
        if block < 16 or block % 16:
            raise ValueError("a cache block holds a multiple of 16 tokens")
        self.fmt, self.block, self.requests = fmt, block, requests
        self.width = -(-capacity // block)
        self.blocks = requests * self.width if blocks is None else blocks
        if self.blocks < 1:
            raise ValueError("the cache needs at least one block")
        dev = torch.device(device)
        shape, scales = (layers, self.blocks, kv_heads, block, head_dim), (layers, self.blocks, kv_heads)
        dtype = ops.FORMATS[fmt]
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device=dev).view(dtype) for _ in range(2))
        self.k_scale, self.v_scale = (torch.ones(scales, device=dev) for _ in range(2))
        self.block_table = torch.empty(requests, self.width, dtype=torch.int32, device=dev)
        self.free_blocks = torch.empty(self.blocks, dtype=torch.int32, device=dev)
        self.state = torch.empty(1 + requests, dtype=torch.int32, device=dev)
        self.clear()

    def clear(self) -> None:
        """All blocks free, all requests empty."""
        self.block_table.fill_(-1)
        self.free_blocks.copy_(torch.arange(self.blocks, dtype=torch.int32))
        self.state.zero_()
        self.state[0] = self.blocks

    def blocks_for(self, tokens: int) -> int:
        return -(-tokens // self.block)

    def require(self, tokens: dict, fresh=()) -> None:
        """Raise ``PoolExhausted`` unless the pool has the blocks for ``tokens[row]`` tokens of each row, beside what all rows
        hold (those in ``fresh`` as if they held none). Where the pool is smaller than all full contexts this reads the
        device."""
        most = max(tokens.values(), default=0)
        if self.blocks_for(most) > self.width:
            raise PoolExhausted(f"{most} tokens need {self.blocks_for(most)} cache blocks, a request has at most {self.width}")
        if self.blocks >= self.requests * self.width:
            return
        held = [0 if row in fresh else n for row, n in enumerate(self.state[1:].tolist())]
        need = sum(max(held[row], self.blocks_for(tokens.get(row, 0))) for row in range(self.requests))
        if need > self.blocks:
            raise PoolExhausted(f"the requests need {need} cache blocks, the pool has {self.blocks}")

    def plan(self, cached_lens: Tensor, new_lens: Tensor, tokens: int) -> ops.BlockPlan:
        """Blocks for the step's new tokens (``ops.plan_blocks``), taken from the pool."""
        plan = ops.plan_blocks(cached_lens, new_lens, self.state, self.block_table, self.free_blocks, self.block, tokens)
        self.state.copy_(plan.state)
        return plan

    def release(self, keep_lens: Tensor) -> None:
        """Give back what lies past each request's first ``keep_lens`` tokens (0: all, -1: nothing)."""
        ops.release_blocks(keep_lens, self.state, self.block_table, self.free_blocks, self.block)

    def release_rows(self, rows) -> None:
        keep = torch.full((self.requests,), -1, dtype=torch.int32)
        keep[rows] = 0
        self.release(keep.to(self.state.device))

    def append(self, layer: int, k: Tensor, v: Tensor, plan: ops.BlockPlan) -> None:
        ops.append_kv(k, v, plan.slot_map, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])

    def attend(self, layer: int, q: Tensor, plan: ops.BlockPlan, max_query: int, max_context: int) -> Tensor:
        return ops.cached_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                    self.block_table, plan.context_lens, plan.query_start, max_query, max_context)
