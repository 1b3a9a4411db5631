"""A block-wise KV cache in 8 bits: its plan, its quantising write and the attention that reads it.

Layout. ``k_cache`` and ``v_cache`` are ``[blocks, kv_heads, block, head_dim]`` in ``float8_e4m3fn`` or ``int8``;
``k_scale`` and ``v_scale`` are float32 ``[blocks, kv_heads]``. A stored number is ``code * scale``; a scale is a power of
two that grows with the block's largest magnitude. Token ``j`` of request ``b`` lies in block
``block_table[b, j // block]``; a *slot* is ``block id * block + j % block``, -1 for none.

One step of a server, all on the device and without a host synchronisation (so that it can be captured):

    plan = plan_blocks(cached_lens, new_lens, state, block_table, free_blocks, block, tokens)
    append_kv(k, v, plan.slot_map, k_cache, v_cache, k_scale, v_scale)                     # every layer
    o = cached_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, plan.context_lens, plan.query_start,
                         max_query, max_context)                                            # every layer

None of it has a backward pass: inputs that ask for gradients are refused.

CUDA tensors go to the sm_100a kernels (``csrc/kv_cache.cu``, ``csrc/cached_attention*.cu``); CPU tensors to the plain
PyTorch forms below. ``inference.paged_cache.PagedKVCache`` holds the storage.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import ext, refuse_gradients

FORMATS = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
_LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
MIN_EXPONENT = -64


class BlockPlan(NamedTuple):
    query_start: Tensor   # int32 [requests + 1]: a request's new tokens are rows [query_start[b], query_start[b + 1])
    context_lens: Tensor  # int32 [requests]: cached and new tokens
    positions: Tensor     # int32 [tokens]; 0 for padding
    slot_map: Tensor      # int32 [tokens]; -1 for padding and for tokens without a block
    state: Tensor         # int32 [1 + requests]: free blocks left, blocks held per request
    missing: Tensor       # int32 [1]: blocks that were needed but not free (or beyond the table's width)


def plan_blocks(cached_lens: Tensor, new_lens: Tensor, state: Tensor, block_table: Tensor, free_blocks: Tensor,
                block: int, tokens: int) -> BlockPlan:
    """Blocks, slots and positions for ``new_lens`` further tokens of each request.

    ``state`` is int32 ``[1 + requests]``: how many of ``free_blocks`` are free (its first entries), then the blocks that
    each request holds already. A request that needs more gets the last free ones, requests in order; their ids go into
    ``block_table`` (in place, from the held entries on). A request without new tokens gets none, whatever its cached
    length. ``state`` itself is left alone: the new one is in the result. ``tokens`` is the number of rows of the step;
    rows past the requests' tokens are padding. Where blocks run out the entries are -1 and ``missing`` counts them."""
    if cached_lens.is_cuda:
        return BlockPlan(*ext().plan_blocks(cached_lens, new_lens, state, block_table, free_blocks, block, tokens))
    cached, new = cached_lens.long().clamp(min=0), new_lens.long().clamp(min=0)
    width = block_table.size(1)
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    wanted = torch.where(new > 0, (cached + new + block - 1) // block, 0)
    fits = wanted.clamp(max=width)
    held = state[1:].long().clamp(min=0, max=width)
    left = min(max(int(state[0]), 0), free_blocks.numel())
    shortage = int((wanted - fits).sum())
    for b in range(cached.numel()):
        for e in range(int(held[b]), int(fits[b])):
            if left > 0:
                left -= 1
                block_table[b, e] = free_blocks[left]
                held[b] += 1
            else:
                block_table[b, e] = -1
                shortage += 1
    positions = torch.zeros(tokens, dtype=torch.int32)
    slots = torch.full((tokens,), -1, dtype=torch.int32)
    for b in range(cached.numel()):
        for i in range(int(new[b])):
            t, p = int(start[b]) + i, int(cached[b]) + i
            if t >= tokens:
                break
            positions[t] = p
            if p // block < width and block_table[b, p // block] >= 0:
                slots[t] = block_table[b, p // block] * block + p % block
    return BlockPlan(start.int(), (cached + new).int(), positions, slots,
                     torch.cat([torch.tensor([left]), held]).int(), torch.tensor([shortage], dtype=torch.int32))


def release_blocks(keep_lens: Tensor, state: Tensor, block_table: Tensor, free_blocks: Tensor, block: int) -> None:
    """Give the blocks past each request's first ``keep_lens`` tokens back (0: all of them, -1: none). ``state``,
    ``block_table`` and ``free_blocks`` change in place."""
    if keep_lens.is_cuda:
        ext().release_blocks(keep_lens, state, block_table, free_blocks, block)
        return
    for b, keep in enumerate(keep_lens.tolist()):
        held = int(state[1 + b])
        kept = held if keep < 0 else min(held, -(-keep // block))
        for e in range(kept, held):
            free_blocks[int(state[0])] = block_table[b, e]
            state[0] += 1
            block_table[b, e] = -1
        state[1 + b] = kept


def _exponent(amax: Tensor, dtype: torch.dtype) -> Tensor:
    m, x = torch.frexp(amax)
    top, up = math.frexp(_LARGEST[dtype])
    return torch.where(amax > 0, (x - up + (m > top).int()).clamp(min=MIN_EXPONENT), MIN_EXPONENT)


def _power(e: Tensor) -> Tensor:
    return torch.ldexp(torch.ones(e.shape), e)


def _encode(x: Tensor, dtype: torch.dtype) -> Tensor:
    x = x.clamp(-_LARGEST[dtype], _LARGEST[dtype])
    return x.nan_to_num(0.0).round().to(dtype) if dtype == torch.int8 else x.to(dtype)


def append_kv(k: Tensor, v: Tensor, slot_map: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor,
              v_scale: Tensor) -> None:
    """Write new keys and values ``[tokens, kv_heads, head_dim]`` (bfloat16, any token and head stride) into their slots.

    The tokens of one block must be neighbours in ``slot_map`` with ascending slots, as ``plan_blocks`` gives them. A run
    that starts at a block's first slot starts the block anew; otherwise the block's scale stays or grows, and the codes
    it holds move to the larger scale. Infinities are stored as the largest code and set no scale; NaN stays NaN in fp8 and
    becomes 0 in int8. Slots of -1 (and outside the cache) are skipped."""
    if k_cache.is_cuda:
        ext().append_kv(k, v, slot_map, k_cache, v_cache, k_scale, v_scale)
        return
    refuse_gradients("append_kv", k, v)
    block = k_cache.size(2)
    slots = slot_map.tolist()
    t = 0
    while t < len(slots):
        n = 1
        if not 0 <= slots[t] < k_cache.size(0) * block:
            t += 1
            continue
        b, first = slots[t] // block, slots[t] % block
        while t + n < len(slots) and slots[t + n] >= 0 and slots[t + n] // block == b:
            n += 1
        for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
            rows = x[t:t + n].float()
            size = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(dim=(0, 2))
            e = _exponent(size, cache.dtype)
            if first:
                # a held scale stays unless the new tokens need a larger one (none is held: 0, or no number)
                m, o = torch.frexp(scale[b])
                e = torch.where((scale[b] > 0) & scale[b].isfinite(), torch.maximum(e, torch.where(m == 0.5, o - 1, o)), e)
                ratio = scale[b] * _power(-e)
                cache[b, :, :first] = _encode(cache[b, :, :first].float() * ratio[:, None, None], cache.dtype)
            codes = _encode(rows * _power(-e)[None, :, None], cache.dtype)
            cache[b][:, [s % block for s in slots[t:t + n]]] = codes.transpose(0, 1)
            scale[b] = _power(e)
        t += n


def cached_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor,
                     context_lens: Tensor, query_start: Tensor, max_query: Optional[int] = None,
                     max_context: Optional[int] = None, scale: Optional[float] = None,
                     out: Optional[Tensor] = None) -> Tensor:
    """Causal attention of the new tokens ``q [tokens, heads, head_dim]`` (bfloat16) over their requests' cached tokens.

    Request ``b`` has rows ``[query_start[b], query_start[b + 1])`` of ``q``; its ``i``-th new token sees the keys up to
    ``context_lens[b] - new + i``, itself included, so the keys and values of the new tokens are appended before. Query
    heads are a multiple of the kv heads (consecutive heads share one). Rows that see no key, and rows of no request, are
    zero. Keys without a block (-1) are not seen. ``max_query`` and ``max_context`` are upper bounds that the host knows;
    they choose the kernel and the split, never the result's meaning. ``scale`` defaults to ``1 / sqrt(head_dim)``."""
    d = k_cache.size(-1)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if k_cache.is_cuda:
        return ext().cached_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, query_start,
                                      max(q.size(0), 1) if max_query is None else max_query,
                                      block_table.size(1) * k_cache.size(2) if max_context is None else max_context,
                                      scale, out)
    refuse_gradients("cached_attention", q, k_scale, v_scale)
    heads, group = q.size(1), q.size(1) // k_cache.size(1)
    if out is None:
        out = torch.empty_like(q)
    out.zero_()
    block, starts = k_cache.size(2), query_start.tolist()
    for b, context in enumerate(context_lens.tolist()):
        lo, hi = starts[b], starts[b + 1]
        length = min(context, block_table.size(1) * block)
        if hi == lo or length <= 0:
            continue
        ids = block_table[b, : -(-length // block)].long()
        here = (ids >= 0).repeat_interleave(block)[:length]
        at = ids.clamp(min=0)
        k, v = (c.view(torch.uint8)[at].view(c.dtype).float() * s[at][..., None, None]
                for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        k, v = (x.transpose(0, 1).reshape(x.size(1), -1, d)[:, :length].repeat_interleave(group, 0) for x in (k, v))
        j, i = torch.arange(length), torch.arange(hi - lo)
        seen = (j[None, :] <= (context - (hi - lo) + i)[:, None]) & here
        scores = torch.einsum("thd,hjd->htj", q[lo:hi].float(), k) * scale
        scores = scores.masked_fill(~seen, -math.inf)
        probs = torch.where(seen.any(-1)[None, :, None], scores.softmax(-1), 0.0)
        for h in range(heads):
            # a masked value counts as zero even where it is NaN
            row_v = torch.where(seen[:, :, None], v[h][None], 0.0)
            out[lo:hi, h] = torch.einsum("tj,tjd->td", probs[h], row_v).to(out.dtype)
    return out
