"""What a serving step does around the model, case by case: the plan of a block-wise KV cache, the quantising write
into it, the attention that reads it, and the processing of the logits.

``listed()`` gives the measured cases, ``draw(rng)`` further ones of the same ranges, ``prepare(case, seed)`` what a
server holds before the call, and ``run(state)`` makes one call: the framework's operator where ``own`` is true, else
the same result from elementary torch operations in 32 bits. ``exact`` is the definition in 64 bits and ``work`` the
bytes and operations that a call cannot do without.

The cache: ``k_cache`` and ``v_cache`` are ``[blocks, kv_heads, block, head_dim]`` in 8 bits (``fp8``: e4m3, ``int8``),
``k_scale`` and ``v_scale`` ``[blocks, kv_heads]`` hold one power of two per block and head, and a stored number stands
for ``code * scale``. Request ``b`` reads token ``j`` in block ``block_table[b, j // block]``.
"""

import math
import random

import torch

own = False

LARGEST = {"fp8": 448.0, "int8": 127.0}  # the largest code
MIN_EXPONENT = -64                       # of a block's scale
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the plan of one decode step of a full server: every request gets one token, some of them a new block
        {"name": "plan-decode-256", "op": "plan", "batch": 256, "new": 1, "longest": 8192, "block": 64, "lens": 1},
        # the plan of a batch of ragged prompts in small blocks, a few of the slots idle
        {"name": "plan-prompts-64", "op": "plan", "batch": 64, "new": 2048, "longest": 0, "block": 16, "lens": 2},
        # one decode step's new keys and values of 32 requests (grouped-query heads of the mixtral-8x7b preset)
        {"name": "append-decode-32", "op": "append", "batch": 32, "new": 1, "longest": 2048, "kv_heads": 8,
         "head_dim": 128, "block": 64, "format": "fp8", "lens": 3},
        # ragged prompts written at once (the moe-1b-e64 preset's heads), starting inside blocks that hold tokens
        {"name": "append-prompts-int8", "op": "append", "batch": 24, "new": 2048, "longest": 100, "kv_heads": 16,
         "head_dim": 64, "block": 32, "format": "int8", "lens": 4},
        # one user, a short conversation: the smallest decode call, where latency is all there is
        {"name": "attend-decode-1", "op": "attend", "batch": 1, "new": 1, "longest": 600, "even": True, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 64, "format": "fp8", "lens": 5},
        # a full server's decode step: 64 requests of every length up to 16K tokens, some slots idle
        {"name": "attend-decode-64", "op": "attend", "batch": 64, "new": 1, "longest": 16384, "even": False,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 64, "format": "fp8", "lens": 6},
        # decode of the moe-1b-e64 preset: as many key/value heads as query heads, odd lengths, small blocks
        {"name": "attend-decode-32-mha", "op": "attend", "batch": 32, "new": 1, "longest": 2047, "even": False,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "block": 16, "format": "int8", "lens": 7},
        # a few drafted tokens per request, checked in one call
        {"name": "attend-verify-8", "op": "attend", "batch": 8, "new": 5, "longest": 8000, "even": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 32, "format": "int8", "lens": 8},
        # the last 2048-token piece of one long prompt that is read piece by piece
        {"name": "attend-chunk-16k", "op": "attend", "batch": 1, "new": 2048, "longest": 14337, "even": True,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 64, "format": "fp8", "lens": 9},
        # a batch of ragged prompts read from their first token (the moe-1b-e64 preset's heads)
        {"name": "attend-prompts-16", "op": "attend", "batch": 16, "new": 2048, "longest": 0, "even": False,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "block": 64, "format": "int8", "lens": 10},
        # one user's next-token logits with every penalty, the ids outside the tokenizer masked
        {"name": "logits-1x32000", "op": "logits", "rows": 1, "vocab": 32000, "dtype": "fp32", "history": 700,
         "biases": 1, "masks": 1, "lens": 11},
        # a full server's logits: some requests with a bias, some with a grammar's mask, a vocabulary of odd size
        {"name": "logits-256x50257", "op": "logits", "rows": 256, "vocab": 50257, "dtype": "bf16", "history": 4096,
         "biases": 4, "masks": 64, "lens": 12},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logits"])
    lens = rng.randrange(1, 1 << 30)
    if op == "plan":
        prompts = rng.random() < 0.5
        return {"op": op, "batch": _log(rng, 1, 64 if prompts else 512), "new": _log(rng, 2, 2048) if prompts else 1,
                "longest": rng.choice([0, _log(rng, 1, 2000)]) if prompts else _log(rng, 1, 16384),
                "block": rng.choice([16, 32, 64, 128]), "lens": lens}
    if op == "logits":
        return {"op": op, "rows": _log(rng, 1, 256), "vocab": rng.choice([512, 7168, 32000, 50257, 50304]),
                "dtype": rng.choice(["fp32", "bf16"]), "history": _log(rng, 1, 4096), "biases": rng.choice([0, 1, 4]),
                "masks": rng.choice([0, 1, 16]), "lens": lens}
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 16, 64), (16, 16, 128), (4, 4, 32), (4, 2, 32), (8, 1, 64),
                                            (12, 4, 64)])
    shape = {"kv_heads": kv_heads, "head_dim": head_dim, "block": rng.choice([16, 32, 64, 128]),
             "format": rng.choice(["fp8", "int8"]), "lens": lens}
    if op == "append":
        prompts = rng.random() < 0.5
        return {"op": op, "batch": _log(rng, 1, 24 if prompts else 128), "new": _log(rng, 2, 2048) if prompts else 1,
                "longest": _log(rng, 1, 1000), **shape}
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    case = {"op": op, "batch": _log(rng, 1, 64 if kind == "decode" else 16), "new": 1, "longest": _log(rng, 1, 16384),
            "even": rng.random() < 0.3, "heads": heads, **shape}
    if kind == "verify":
        case["new"] = rng.randrange(2, 9)
    if kind == "prompt":
        case.update(new=_log(rng, 9, 2048), longest=rng.choice([0, _log(rng, 1, 14337)]))
    top = max(work(c)["flops"] for c in listed() if c["op"] == "attend")
    while work(case)["flops"] > top or case["batch"] * case["new"] * case["heads"] * (case["longest"] + case["new"]) > 1.1e9:
        case["batch"] = max(1, case["batch"] // 2)
        if case["batch"] == 1:
            case["new"], case["longest"] = max(1, case["new"] * 3 // 4), case["longest"] * 3 // 4
    return case


def lengths(case):
    """[(tokens in the cache before the call, new tokens)] of the case's requests: most within a factor of eight of the
    longest, some of any length, the last the longest. In a large ragged batch every eighth slot is idle: nothing
    cached, nothing new."""
    rng = random.Random(case["lens"])
    batch, new, longest = case["batch"], case["new"], case["longest"]
    if case.get("even"):
        return [(longest, new)] * batch
    got = []
    for i in range(batch):
        if batch >= 16 and i % 8 == 5:
            got.append((0, 0))
        elif i == batch - 1:
            got.append((longest, new))
        else:
            got.append((_log(rng, max(1, longest // 8) if i % 4 else 1, longest) if longest else 0,
                        _log(rng, max(1, new // 16), new)))
    return got


def work(case):
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        b = 2 * n * size + case["rows"] * (case["history"] * 4 + 28) + min(case["biases"], case["rows"]) * case["vocab"] * 4
        b += min(case["masks"], case["rows"]) * ((case["vocab"] + 31) // 32) * 4
        return {"bytes": b, "flops": 4 * n}
    lens, block = lengths(case), case["block"]
    tokens = sum(n for _, n in lens)
    if case["op"] == "plan":
        fresh = sum(-(-(c + n) // block) - -(-c // block) for c, n in lens)
        return {"bytes": 8 * tokens + 24 * len(lens) + 8 * fresh, "flops": 0}
    hkv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        blocks = sum(-(-(c + n) // block) - c // block for c, n in lens if n)
        return {"bytes": tokens * (hkv * d * 2 * (2 + 1) + 4) + blocks * hkv * 2 * 4, "flops": 4 * tokens * hkv * d}
    heads = case["heads"]
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in lens)
    read = sum((c + n) * 2 * hkv * d + -(-(c + n) // block) * (2 * hkv * 4 + 4) for c, n in lens if n)
    return {"bytes": read + 2 * tokens * heads * d * 2, "flops": 4 * pairs * heads * d}


# --------------------------------------------------------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lens):
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    return starts


def _quantised(x, fmt):
    """Codes and scales of ``x [blocks, heads, block, dim]``, as a cache holds them."""
    amax = x.abs().amax(dim=(2, 3)).float()
    scale = torch.ldexp(torch.ones_like(amax), torch.ceil(torch.log2(amax / LARGEST[fmt])).int())
    codes = x.float() / scale[:, :, None, None]
    codes = codes.clamp(-LARGEST[fmt], LARGEST[fmt])
    return (codes.round() if fmt == "int8" else codes).to(CODES[fmt]), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "logits":
        return _prepare_logits(case, g)
    lens, block = lengths(case), case["block"]
    batch, tokens = len(lens), sum(n for _, n in lens)
    held = [-(-c // block) for c, _ in lens]
    need = [-(-(c + n) // block) for c, n in lens]
    width = max(max(need), 1) + 2
    blocks = sum(need) + 16
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    # a table whose first entries of each request are taken; a plan's request still gets the others
    taken = held if op == "plan" else need
    at = torch.cumsum(_ints([0] + taken[:-1]), 0)
    column = torch.arange(width, device="cuda")
    table = torch.where(column < _ints(taken)[:, None], order[(at[:, None] + column).clamp(max=blocks - 1)], -1).to(torch.int32)
    state = {"op": op, "block": block, "tokens": tokens, "block_table": table,
             "cached_lens": _ints([c for c, _ in lens]), "new_lens": _ints([n for _, n in lens])}
    if op == "plan":
        free = order[sum(held):].contiguous()
        state.update(free_blocks=free, state=_ints([free.numel()] + held))
        return state
    hkv, d, fmt = case["kv_heads"], case["head_dim"], case["format"]
    state.update(format=fmt, query_start=_ints(_starts(lens)), context_lens=_ints([c + n for c, n in lens]))

    def cache():
        # keys and values of a trained model: unlike sizes of the channels, and a few large ones
        channel = torch.exp(0.5 * torch.randn(1, hkv, 1, d, generator=g, device="cuda"))
        x = torch.randn(blocks, hkv, block, d, generator=g, device="cuda", dtype=torch.bfloat16)
        return _quantised(x * channel.to(torch.bfloat16), fmt)

    state["k_cache"], state["k_scale"] = cache()
    state["v_cache"], state["v_scale"] = cache()
    if op == "append":
        # rows of a packed query/key/value projection: the heads of one token lie together, the tokens apart
        rows = torch.randn(tokens, 3 * hkv, d, generator=g, device="cuda", dtype=torch.bfloat16)
        state["k"], state["v"] = rows[:, hkv:2 * hkv], rows[:, 2 * hkv:]
        request = torch.repeat_interleave(torch.arange(batch, device="cuda"), state["new_lens"].long())
        position = torch.arange(tokens, device="cuda") - state["query_start"][request] + state["cached_lens"][request]
        state["slot_map"] = (table[request, position // block] * block + position % block).to(torch.int32)
        return state
    state["q"] = torch.randn(tokens, case["heads"], d, generator=g, device="cuda", dtype=torch.bfloat16)
    state["max_query"] = max(n for _, n in lens)
    state["max_context"] = max(c + n for c, n in lens)
    return state


def _prepare_logits(case, g):
    rows, vocab, length = case["rows"], case["vocab"], case["history"]
    rng = random.Random(case["lens"])
    used = [_log(rng, 1, length) for _ in range(rows - 1)] + [length]
    prompt = [rng.randrange(0, n + 1) for n in used]
    # token ids as texts have them: a few very often
    u = torch.rand(rows, length, generator=g, device="cuda")
    history = torch.exp(u * math.log(vocab)).long().clamp(max=vocab) - 1
    some = lambda low, high: torch.rand(rows, generator=g, device="cuda") * (high - low) + low  # noqa: E731
    state = {"op": "logits", "history": history.to(torch.int32), "history_lens": _ints(used), "prompt_lens": _ints(prompt),
             "logits": (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(DTYPES[case["dtype"]]),
             "repetition": some(1.0, 1.5), "frequency": some(0.0, 0.5), "presence": some(0.0, 0.8),
             "bias": None, "bias_rows": None, "mask": None, "mask_rows": None}
    if case["biases"]:
        few = torch.rand(case["biases"], vocab, generator=g, device="cuda") < 0.01
        state["bias"] = torch.randn(case["biases"], vocab, generator=g, device="cuda") * few
        state["bias_rows"] = torch.arange(rows, device="cuda", dtype=torch.int32) % (2 * case["biases"])
        state["bias_rows"][state["bias_rows"] >= case["biases"]] = -1 if rows > 1 else 0
    if case["masks"]:
        words = (vocab + 31) // 32
        state["mask"] = torch.randint(-(1 << 31), (1 << 31) - 1, (case["masks"], words), generator=g, device="cuda").to(torch.int32)
        state["mask_rows"] = torch.arange(rows, device="cuda", dtype=torch.int32) % (2 * case["masks"])
        state["mask_rows"][state["mask_rows"] >= case["masks"]] = -1 if rows > 1 else 0
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[s["op"]](s)


def _own(s):
    from quantaweave_b200.ops import kv_cache
    from quantaweave_b200.ops.logits import process_logits

    if s["op"] == "plan":
        p = kv_cache.plan_blocks(s["cached_lens"], s["new_lens"], s["state"], s["block_table"], s["free_blocks"], s["block"],
                                 s["tokens"])
        return {"query_start": p.query_start, "context_lens": p.context_lens, "positions": p.positions,
                "slot_map": p.slot_map, "state": p.state, "missing": p.missing, "block_table": s["block_table"]}
    if s["op"] == "append":
        kv_cache.append_kv(s["k"], s["v"], s["slot_map"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["op"] == "attend":
        return kv_cache.cached_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                         s["context_lens"], s["query_start"], s["max_query"], s["max_context"])
    return process_logits(s["logits"], history=s["history"], history_lens=s["history_lens"], prompt_lens=s["prompt_lens"],
                          repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias=s["bias"],
                          bias_rows=s["bias_rows"], mask=s["mask"], mask_rows=s["mask_rows"])


def _plain_plan(s):
    cached, new, table, block, tokens = s["cached_lens"], s["new_lens"], s["block_table"], s["block"], s["tokens"]
    free_blocks, free, held = s["free_blocks"], s["state"][:1], s["state"][1:]
    width, dev = table.size(1), table.device
    ends = torch.cumsum(new, 0, dtype=torch.int32)
    query_start = torch.cat([ends.new_zeros(1), ends])
    context = cached + new
    wanted = (context + block - 1) // block
    fits = wanted.clamp(max=width)
    grow = (fits - held).clamp(min=0)
    rank_end = torch.cumsum(grow, 0, dtype=torch.int32)
    rank_start = rank_end - grow
    # the table: request b's new entries are the next free blocks, taken from the end of the list
    column = torch.arange(width, device=dev, dtype=torch.int32)
    is_new = (column >= held[:, None]) & (column < fits[:, None])
    rank = rank_start[:, None] + column - held[:, None]
    there = rank < free
    block_id = free_blocks[(free - 1 - rank).clamp(min=0, max=free_blocks.numel() - 1).long()]
    table.copy_(torch.where(is_new, torch.where(there, block_id, -1), table))
    got = (free - rank_start).clamp(min=0)
    given = torch.minimum(grow, got)
    taken = torch.minimum(rank_end[-1:], free)
    state = torch.cat([free - taken, held + given])
    missing = (rank_end[-1:] - taken) + (wanted - fits).clamp(min=0).sum(dtype=torch.int32)
    t = torch.arange(tokens, device=dev, dtype=torch.int32)
    request = (t[:, None] >= ends[None, :]).sum(1).clamp(max=new.numel() - 1)
    real = t < ends[-1]
    position = torch.where(real, t - query_start[request] + cached[request], 0)
    entry = position // block
    where = table[request, entry.clamp(max=width - 1)]
    slot = torch.where(real & (entry < width) & (where >= 0), where * block + position % block, -1)
    return {"query_start": query_start, "context_lens": context, "positions": position, "slot_map": slot, "state": state,
            "missing": missing.to(torch.int32), "block_table": table}


def _exponent(amax, fmt):
    """The least e with amax <= largest code * 2^e, in 32 bits."""
    m, x = torch.frexp(amax)
    top, up = math.frexp(LARGEST[fmt])
    e = x - up + (m > top).to(torch.int32)
    return torch.where(amax > 0, e.clamp(min=MIN_EXPONENT), MIN_EXPONENT)


def _codes(x, fmt):
    x = x.clamp(-LARGEST[fmt], LARGEST[fmt])
    return x.round().to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)


def _plain_append_one(x, cache, scales, slot, block, fmt):
    x = x.float()
    unit = torch.ones((), device=x.device)
    touched, which = torch.unique(slot // block, return_inverse=True)
    offset = slot % block
    first = torch.full_like(touched, block).scatter_reduce(0, which, offset, "amin")
    size = x.abs().amax(-1)
    amax = torch.zeros(touched.numel(), x.size(1), device=x.device)
    amax = amax.scatter_reduce(0, which[:, None].expand_as(size), size, "amax")
    fresh = _exponent(amax, fmt)
    old = torch.frexp(scales[touched])[1] - 1
    exponent = torch.where((first > 0)[:, None], torch.maximum(old, fresh), fresh)
    # what the blocks held before, on the new scale
    rows = cache.view(torch.uint8)[touched].view(cache.dtype)
    again = _codes(rows.float() * torch.ldexp(unit, (old - exponent))[:, :, None, None], fmt)
    keep = (torch.arange(block, device=x.device) < first[:, None])[:, None, :, None]
    rows = torch.where(keep, again.view(torch.uint8), rows.view(torch.uint8))
    codes = _codes(x * torch.ldexp(unit, -exponent[which])[:, :, None], fmt)
    rows[which, :, offset] = codes.view(torch.uint8)
    cache.view(torch.uint8)[touched] = rows
    scales[touched] = torch.ldexp(unit, exponent)


def _plain_append(s):
    slot = s["slot_map"].long()
    _plain_append_one(s["k"], s["k_cache"], s["k_scale"], slot, s["block"], s["format"])
    _plain_append_one(s["v"], s["v_cache"], s["v_scale"], slot, s["block"], s["format"])
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gathered(cache, scale, table, length):
    """``[batch, kv_heads, length, dim]`` in 32 bits: the blocks of each request in their order."""
    at = table[:, : -(-length // cache.size(2))].clamp(min=0).long()
    x = cache.view(torch.uint8)[at].view(cache.dtype).float() * scale[at][..., None, None]
    batch, n, heads, block, dim = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(batch, heads, n * block, dim)[:, :, :length]


def _plain_attend(s):
    q, start, context = s["q"], s["query_start"].long(), s["context_lens"].long()
    tokens, heads, dim = q.shape
    longest, most = s["max_context"], s["max_query"]
    k = _gathered(s["k_cache"], s["k_scale"], s["block_table"], longest)
    v = _gathered(s["v_cache"], s["v_scale"], s["block_table"], longest)
    batch, kv_heads = k.size(0), k.size(1)
    new = start[1:] - start[:-1]
    i = torch.arange(most, device=q.device)
    at = (start[:-1, None] + i).clamp(max=tokens - 1)
    qs = q[at].float().view(batch, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    qs = qs.reshape(batch, kv_heads, -1, dim)
    j = torch.arange(longest, device=q.device)
    seen = (j <= (context - new)[:, None, None] + i[:, None]) & (i < new[:, None])[..., None]
    there = (j < context[:, None])[:, None, :, None]
    scores = torch.matmul(qs, torch.where(there, k, 0.0).transpose(-1, -2)) / math.sqrt(dim)
    scores = scores.view(batch, kv_heads, heads // kv_heads, most, longest).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(batch, kv_heads, -1, longest), torch.where(there, v, 0.0)).view(*e.shape[:-1], dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    t = torch.arange(tokens, device=q.device)
    request = (t[:, None] >= start[None, 1:]).sum(1).clamp(max=batch - 1)
    return o[request, t - start[request]].to(q.dtype)


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(s["history"].size(1), device=x.device)
    used = at < s["history_lens"][:, None]
    made = used & (at >= s["prompt_lens"][:, None])
    ids = s["history"].long()
    seen = torch.zeros_like(x).scatter_add(1, ids, used.float())
    count = torch.zeros_like(x).scatter_add(1, ids, made.float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - count * s["frequency"][:, None] - (count > 0).float() * s["presence"][:, None]
    if s["bias"] is not None:
        has = s["bias_rows"] >= 0
        x = torch.where(has[:, None], x + s["bias"][s["bias_rows"].clamp(min=0).long()], x)
    if s["mask"] is not None:
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        bit = (words[..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        free = bit.reshape(rows, -1)[:, :vocab].bool() | (s["mask_rows"] < 0)[:, None]
        x = torch.where(free, x, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "logits":
        return _exact_logits(s)
    return None  # whole numbers


def _exact_append(s):
    fmt, block, slots = s["format"], s["block"], s["slot_map"].tolist()
    runs, at = [], 0  # (block, first token, tokens): the tokens of one block are next to one another
    for t in range(1, len(slots) + 1):
        if t == len(slots) or slots[t] // block != slots[at] // block:
            runs.append((slots[at] // block, at, t - at))
            at = t

    def power(e):
        return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)

    def onto_codes(x):
        x = x.clamp(-LARGEST[fmt], LARGEST[fmt])
        if fmt == "int8":
            return x.round()
        step = power((torch.frexp(x)[1] - 1).clamp(min=-6) - 3)  # of the numbers with 4 significant bits, from 2^-9 on
        return torch.round(x / step) * step

    def one(x, cache, scales):
        x, held, scales = x.double(), cache.double(), scales.double()
        amax = x.abs().amax(-1)
        for b, t, n in runs:
            first = slots[t] % block
            top = amax[t:t + n].amax(0)
            part, e = torch.frexp(top / LARGEST[fmt])
            unit = power((e - (part == 0.5).int()).clamp(min=MIN_EXPONENT))
            if first:
                unit = torch.maximum(unit, scales[b])
                held[b, :, :first] = onto_codes(held[b, :, :first] * (scales[b] / unit)[:, None, None])
            held[b, :, first:first + n] = onto_codes(x[t:t + n].transpose(0, 1) / unit[:, None, None])
            scales[b] = unit
        return held, scales

    k, ks = one(s["k"], s["k_cache"], s["k_scale"])
    v, vs = one(s["v"], s["v_cache"], s["v_scale"])
    whole = fmt == "int8"
    return {"k": None if whole else k, "v": None if whole else v, "k_scale": ks, "v_scale": vs}


def _exact_attend(s):
    q = s["q"].double()
    heads, dim = q.size(1), q.size(2)
    out = torch.zeros_like(q)
    starts, context, block = s["query_start"].tolist(), s["context_lens"].tolist(), s["block"]
    for b, total in enumerate(context):
        lo, hi = starts[b], starts[b + 1]
        if hi == lo:
            continue
        at = s["block_table"][b, : -(-total // block)].long()

        def read(cache, scale):
            x = cache.view(torch.uint8)[at].view(cache.dtype).double() * scale[at].double()[..., None, None]
            return x.transpose(0, 1).reshape(x.size(1), -1, dim)[:, :total]

        k, v = read(s["k_cache"], s["k_scale"]), read(s["v_cache"], s["v_scale"])
        group = heads // k.size(0)
        last = total - (hi - lo) + torch.arange(hi - lo, device=q.device)
        hidden = torch.arange(total, device=q.device) > last[:, None]
        for h in range(heads):
            scores = (q[lo:hi, h] @ k[h // group].T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            out[lo:hi, h] = torch.softmax(scores, -1) @ v[h // group]
    return out


def _exact_logits(s):
    x = s["logits"].double()
    vocab = x.size(1)
    used, prompt = s["history_lens"].tolist(), s["prompt_lens"].tolist()
    for r in range(x.size(0)):
        ids = s["history"][r, : used[r]].long()
        seen = torch.bincount(ids, minlength=vocab) > 0
        made = torch.bincount(ids[prompt[r]:], minlength=vocab).double()
        factor = s["repetition"][r].double()
        y = torch.where(seen, torch.where(x[r] > 0, x[r] / factor, x[r] * factor), x[r])
        y = y - made * s["frequency"][r].double() - (made > 0) * s["presence"][r].double()
        if s["bias"] is not None and int(s["bias_rows"][r]) >= 0:
            y = y + s["bias"][int(s["bias_rows"][r])].double()
        if s["mask"] is not None and int(s["mask_rows"][r]) >= 0:
            words = s["mask"][int(s["mask_rows"][r])].long() & 0xFFFFFFFF
            id_ = torch.arange(vocab, device=x.device)
            y = y.masked_fill((words[id_ // 32] >> (id_ % 32)) & 1 == 0, -math.inf)
        x[r] = y
    return x
