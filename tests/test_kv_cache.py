"""The block-wise 8-bit KV cache: plan, release, quantising write and attention against definitions in 64 bits, on the
CPU path and on the sm_100a kernels.

Tolerances. Codes, scales and everything whole are exact: a scale is a power of two, so a code is one correctly rounded
number. The attention kernels round the probabilities to f16 (2^-11 relative, each) and the result to bf16 (2^-9 of it);
scores and sums are in 32 bits, ex2 is good to 2^-22. Below 2^-14 an f16 weight is a multiple of 2^-24; a weight is the
probability over the running largest one, times 2^8, times the value's scale over the largest, so the absolute error of one
key's part is at most 2^-33 times the largest scale times its code. So |error| <= 2^-8 |o| + 2^-10 sum_j p_j |v_j| +
2^-32 max_j scale_j sum_j |code_j| holds with a factor of two to spare on each term."""

import math
import sys

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200.ops import kv_cache as kvc

DEVICES = ["cpu", pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")])]
LARGEST = {"fp8": 448.0, "int8": 127.0}


# ------------------------------------------------------------------------------------------------------------ plan
def _pool(held, blocks, width, seed=0):
    """(state, table, free list) of requests that hold ``held`` blocks each of a pool of ``blocks``."""
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(held), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = torch.cat([order[at:], torch.full((at,), -1, dtype=torch.int32)])
    return torch.tensor([blocks - at] + list(held), dtype=torch.int32), table, free


def _plan_oracle(cached, new, state, table, free, block, tokens):
    table, left, held = table.clone(), int(state[0]), state[1:].tolist()
    missing, starts, positions, slots = 0, [0], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        want = -(-(c + n) // block)
        for e in range(held[b], want):
            if e >= table.size(1):
                missing += 1
            elif left > 0:
                left -= 1
                table[b, e] = free[left]
                held[b] += 1
            else:
                table[b, e] = -1
                missing += 1
        for p in range(c, c + n):
            positions.append(p)
            e = p // block
            slots.append(int(table[b, e]) * block + p % block if e < table.size(1) and table[b, e] >= 0 else -1)
        starts.append(starts[-1] + n)
    pad = tokens - len(positions)
    return starts, positions[:tokens] + [0] * pad, slots[:tokens] + [-1] * pad, [left] + held, missing, table


PLANS = {
    "one token": ([0], [1], 16, 4, 8, 0),
    "nothing": ([0, 0, 5], [0, 0, 0], 16, 8, 8, 0),
    "decode at block ends": ([15, 16, 17, 31, 32, 0], [1] * 6, 16, 40, 4, 0),
    "ragged prompts": ([0, 7, 0, 100, 3], [33, 1, 0, 70, 200], 32, 40, 16, 0),
    "padding rows": ([4, 9], [3, 2], 16, 9, 4, 7),
    "pool runs out": ([0, 10, 0], [40, 30, 50], 16, 5, 8, 0),
    "table too narrow": ([0, 30], [100, 5], 16, 20, 3, 0),
    "many requests": (list(range(0, 900, 3)), [1 + i % 5 for i in range(300)], 64, 5000, 20, 0),
    "long step": ([0, 5], [3000, 2500], 16, 400, 200, 0),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", list(PLANS))
def test_plan_matches_its_definition(case, device):
    cached, new, block, blocks, width, pad = PLANS[case]
    held = [min(-(-c // block), width) for c in cached]
    state, table, free = _pool(held, max(blocks, sum(held)), width)
    tokens = sum(new) + pad
    starts, positions, slots, left, missing, want_table = _plan_oracle(cached, new, state, table, free, block, tokens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got_table, before = table.clone().to(device), state.clone().to(device)
    plan = kvc.plan_blocks(i32(cached), i32(new), before, got_table, free.to(device), block, tokens)
    assert plan.query_start.tolist() == starts
    assert plan.context_lens.tolist() == [c + n for c, n in zip(cached, new)]
    assert plan.positions.tolist() == positions
    assert plan.slot_map.tolist() == slots
    assert plan.state.tolist() == left and plan.missing.tolist() == [missing]
    assert torch.equal(got_table.cpu(), want_table)
    assert torch.equal(before.cpu(), state)  # the caller's state is left alone


@pytest.mark.parametrize("device", DEVICES)
def test_plan_of_a_rewound_request_keeps_its_blocks(device):
    state, table, free = _pool([4, 1], 8, 6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    t = table.clone().to(device)
    plan = kvc.plan_blocks(i32([20, 15]), i32([3, 1]), state.to(device), t, free.to(device), 16, 4)
    assert plan.state.tolist() == state.tolist() and torch.equal(t.cpu(), table)
    assert plan.slot_map.tolist() == [int(table[0, 1]) * 16 + 4 + i for i in range(3)] + [int(table[1, 0]) * 16 + 15]


@pytest.mark.parametrize("device", DEVICES)
def test_released_blocks_return_and_are_given_again(device):
    state, table, free = _pool([3, 0, 2, 5], 16, 6)
    s, t, f = (x.clone().to(device) for x in (state, table, free))
    kvc.release_blocks(torch.tensor([17, 4, -1, 0], dtype=torch.int32, device=device), s, t, f, 16)
    assert s.tolist() == [16 - 10 + 1 + 5, 2, 0, 2, 0]
    assert t[0].tolist() == table[0, :2].tolist() + [-1] * 4 and t[2].tolist() == table[2].tolist()
    assert t[3].tolist() == [-1] * 6
    assert f[6:12].tolist() == [int(table[0, 2])] + table[3, :5].tolist()
    held = set(t[t >= 0].tolist())
    assert held.isdisjoint(f[:12].tolist()) and len(held | set(f[:12].tolist())) == 16  # no block lost or doubled


# ---------------------------------------------------------------------------------------------------------- append
def _round_codes(x, fmt):
    """x (float64, on the scale) to the nearest code, ties to even."""
    x = x.clamp(-LARGEST[fmt], LARGEST[fmt])
    if fmt == "int8":
        return torch.nan_to_num(x, nan=0.0).round()
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.where(x.isnan(), x, (x / step).round() * step)


def _append_oracle(x, slots, codes, scale, fmt):
    codes, scale = codes.double(), scale.double()
    block = codes.size(2)
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < codes.size(0) * block:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] // block == slots[t] // block and slots[t + n] >= 0:
            n += 1
        b, first = slots[t] // block, slots[t] % block
        for h in range(codes.size(1)):
            rows = x[t:t + n, h].double()
            size = rows[rows.isfinite()].abs().max().item() if rows.isfinite().any() else 0.0
            unit = 2.0 ** -64
            while size > LARGEST[fmt] * unit:
                unit *= 2
            if first:
                unit = max(unit, scale[b, h].item())
                codes[b, h, :first] = _round_codes(codes[b, h, :first] * (scale[b, h].item() / unit), fmt)
            for i in range(n):
                codes[b, h, slots[t + i] % block] = _round_codes(rows[i] / unit, fmt)
            scale[b, h] = unit
        t += n
    return codes, scale


def _same(got, want):
    return torch.equal(torch.nan_to_num(got, nan=1e30), torch.nan_to_num(want, nan=1e30))


APPENDS = [  # slots' runs as (block, first, tokens) or -1 (padding), kv heads, head_dim, tokens of a block
    ([(2, 0, 1)], 1, 64, 16),
    ([(0, 5, 1), (3, 15, 1), -1, (1, 0, 1), (2, 9, 1)], 3, 128, 16),
    ([(4, 3, 13), (1, 0, 16), (6, 0, 7)], 2, 32, 16),
    ([-1, (0, 60, 4), (5, 0, 64), (2, 0, 64), (1, 0, 1), -1], 2, 128, 64),
    ([(1, 1, 127), (0, 0, 128), (2, 0, 30)], 1, 128, 128),
    ([(i, (7 * i) % 32, 1) for i in range(40)], 5, 64, 32),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_writes_codes_and_scales(case, fmt, device):
    runs, heads, dim, block = APPENDS[case]
    g = torch.Generator().manual_seed(case)
    slots = []
    for r in runs:
        slots += [-1] if r == -1 else [r[0] * block + r[1] + i for i in range(r[2])]
    blocks, tokens = 1 + max(s // block for s in slots), len(slots)
    big = torch.exp2(torch.randint(-6, 7, (tokens, heads, 1), generator=g).float())  # scales have to grow, and not to
    rows = (torch.randn(tokens, 3 * heads, dim, generator=g) * torch.cat([big, big, 1 / big], 1)).bfloat16()
    held = torch.randint(-127, 128, (2, blocks, heads, block, dim), generator=g)
    codes = held.to(torch.int8) if fmt == "int8" else held.float().to(torch.float8_e4m3fn)
    scale = torch.exp2(torch.randint(-9, 3, (2, blocks, heads), generator=g).float())
    rows_d = rows.to(device)
    k, v = rows_d[:, heads:2 * heads], rows_d[:, 2 * heads:]  # rows of a packed projection
    kc, vc, ks, vs = (x.clone().to(device) for x in (codes[0], codes[1], scale[0], scale[1]))
    kvc.append_kv(k, v, torch.tensor(slots, dtype=torch.int32, device=device), kc, vc, ks, vs)
    for x, c, s, i in ((k, kc, ks, 0), (v, vc, vs, 1)):
        want_c, want_s = _append_oracle(x.cpu(), slots, codes[i], scale[i], fmt)
        assert _same(s.double().cpu(), want_s)
        assert _same(c.cpu().double(), want_c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_append_of_zeros_infinities_and_nan(fmt, device):
    x = torch.randn(6, 2, 32, generator=torch.Generator().manual_seed(0))
    x[0] = 0.0                      # a block of zeros only
    x[2, 0, 3], x[2, 1, 4] = math.inf, -math.inf
    x[3, 0, 5] = math.nan
    x[4] = 1e-30                    # below the least scale
    x[5] = 3e38
    x = x.bfloat16()
    slots = [0, 16, 17, 18, 40, 48]
    codes = torch.zeros(4, 2, 16, 32, dtype=kvc.FORMATS[fmt])
    scale = torch.ones(4, 2)
    kc, vc, ks, vs = (t.clone().to(device) for t in (codes, codes, scale, scale))
    kvc.append_kv(x.to(device), (-x).to(device), torch.tensor(slots, dtype=torch.int32, device=device), kc, vc, ks, vs)
    for y, c, s in ((x, kc, ks), (-x, vc, vs)):
        want_c, want_s = _append_oracle(y, slots, codes, scale, fmt)
        assert _same(s.double().cpu(), want_s) and _same(c.cpu().double(), want_c)
    assert kc.cpu().float()[1, 0, 1, 3] == LARGEST[fmt] and kc.cpu().float()[1, 1, 1, 4] == -LARGEST[fmt]


@pytest.mark.parametrize("device", DEVICES)
def test_append_takes_any_stride_and_offset(device):
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(3 + 9 * 2 * 64, generator=g).bfloat16().to(device)
    odd = flat[3:].view(9, 2, 64)                                        # not on a 16-byte boundary
    turned = torch.randn(2, 64, 9, generator=g).bfloat16().to(device).permute(2, 0, 1)  # head_dim not innermost
    both = torch.zeros(4, 2, 2, 16, 64, dtype=torch.int8, device=device)  # keys and values of a block side by side
    scale = torch.zeros(4, 2, 2, device=device)
    slots = torch.tensor([33, 34, 35, 36, 37, 38, 39, 40, 41], dtype=torch.int32, device=device) - 1
    kvc.append_kv(odd, turned, slots, both[:, 0], both[:, 1], scale[:, 0], scale[:, 1])
    for i, x in enumerate((odd, turned)):
        want_c, want_s = _append_oracle(x.cpu(), slots.tolist(), torch.zeros(4, 2, 16, 64, dtype=torch.int8),
                                        torch.zeros(4, 2), "int8")
        assert torch.equal(both[:, i].cpu().double(), want_c) and torch.equal(scale[:, i].cpu().double(), want_s)


# ------------------------------------------------------------------------------------------------------- attention
def _attend_oracle(q, kc, vc, ks, vs, table, context, starts, scale):
    """(o, its tolerance) in 64 bits."""
    q = q.double().cpu()
    kc, vc, ks, vs, table = (t.cpu() for t in (kc, vc, ks, vs, table))
    k_all, v_all = kc.double() * ks.double()[..., None, None], vc.double() * vs.double()[..., None, None]
    codes = vc.double().abs()
    heads, group, block = q.size(1), q.size(1) // kc.size(1), kc.size(2)
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    for b, ctx in enumerate(context):
        n = starts[b + 1] - starts[b]
        j = [j for j in range(min(ctx, table.size(1) * block)) if table[b, j // block] >= 0]
        if not j or not n:
            continue
        pages, offs = table[b].long()[[i // block for i in j]], torch.tensor([i % block for i in j])
        k, v, c = k_all[pages, :, offs], v_all[pages, :, offs], codes[pages, :, offs]  # [keys, kv heads, dim]
        where = torch.tensor(j)
        for i in range(n):
            seen = where <= ctx - n + i
            if not seen.any():
                continue
            for h in range(heads):
                s = (k[seen][:, h // group] @ q[starts[b] + i, h]) * scale
                p = (s - s.max()).exp()
                p = p / p.sum()
                o[starts[b] + i, h] = p @ v[seen][:, h // group]
                top = vs[pages][seen][:, h // group].double().max()
                size[starts[b] + i, h] = (2.0 ** -8 * o[starts[b] + i, h].abs() + 2.0 ** -10 * (p @ v[seen][:, h // group].abs())
                                          + 2.0 ** -32 * top * c[seen][:, h // group].sum(0))
    return o, size


def _cache(blocks, heads, block, dim, fmt, g):
    out = []
    for _ in range(2):
        x = torch.randn(blocks, heads, block, dim, generator=g) * torch.exp2(torch.randint(-3, 4, (blocks, heads, 1, 1), generator=g).float())
        amax = x.abs().amax((2, 3))
        scale = torch.exp2(torch.ceil(torch.log2(amax / LARGEST[fmt])))
        codes = x / scale[..., None, None]
        out += [codes.round().to(torch.int8) if fmt == "int8" else codes.to(torch.float8_e4m3fn), scale]
    return out[0], out[2], out[1], out[3]


def _requests(lens, block, g, spare=3):
    """(table, context, query starts, blocks) for [(cached, new)]."""
    need = [-(-(c + n) // block) for c, n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=g).int()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at, starts = 0, [0]
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        starts.append(starts[-1] + lens[b][1])
    return table, [c + n for c, n in lens], starts, blocks


def _check(o, want, size):
    o = o.double().cpu()
    assert torch.isfinite(o).all()
    over = (o - want).abs() - size - 1e-30
    assert over.max() <= 0, over.max().item()


SHAPES = [  # [(cached, new)], heads, kv heads, head_dim, block
    ([(0, 1)], 4, 4, 64, 16),                                  # the very first token
    ([(1, 1), (15, 1), (16, 1), (63, 1), (64, 1)], 4, 2, 32, 16),
    ([(100, 1), (0, 0), (777, 1), (5, 0), (0, 1)], 8, 2, 128, 64),  # idle slots between
    ([(1500, 1)], 8, 1, 128, 32),                              # one long request: split over all blocks
    ([(300, 3), (40, 8), (0, 5)], 12, 4, 64, 32),              # drafted tokens, three heads to a kv head
    ([(129, 2)], 32, 1, 64, 128),                              # 32 heads on one kv head
    ([(0, 77), (50, 40), (200, 1)], 4, 4, 32, 16),             # prompts
    ([(0, 150), (33, 64), (3, 1)], 4, 2, 64, 16),
    ([(0, 200), (130, 70), (64, 64)], 4, 4, 64, 64),
    ([(0, 130), (700, 40)], 8, 2, 128, 64),
    ([(20, 300)], 6, 2, 128, 16),                              # three heads to a kv head: rows end inside a token
    ([(0, 1)] * 40, 2, 2, 128, 16),                            # many short requests
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_matches_64_bits(case, fmt, device):
    lens, heads, kv_heads, dim, block = SHAPES[case]
    g = torch.Generator().manual_seed(100 + case)
    table, context, starts, blocks = _requests(lens, block, g)
    kc, vc, ks, vs = _cache(blocks, kv_heads, block, dim, fmt, g)
    q = (2 * torch.randn(starts[-1], heads, dim, generator=g)).bfloat16()
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    args = [t.to(device) for t in (q, kc, vc, ks, vs, table)] + [i32(context), i32(starts)]
    bounds = (max(n for _, n in lens), max(context))
    o = kvc.cached_attention(*args, *bounds)
    _check(o, want, size)
    again = kvc.cached_attention(*args, *bounds)
    assert torch.equal(o, again)                      # no order of atomics decides anything
    _check(kvc.cached_attention(*args), want, size)  # loose bounds: another split, the same meaning


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("lens", [[(70, 1), (3, 4)], [(40, 150), (0, 90)]])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_masked_does_not_count(dim, lens, fmt, device):
    """Codes past a request's tokens, blocks that are not there, tokens of no request and rows that see nothing."""
    g = torch.Generator().manual_seed(7)
    block, heads, kv_heads = 32, 4, 2
    table, context, starts, blocks = _requests(lens, block, g)
    kc, vc, ks, vs = _cache(blocks, kv_heads, block, dim, fmt, g)
    table[0, 1] = -1  # a block in the middle that was never given
    for b, ctx in enumerate(context):  # what lies behind the last token: the worst that 8 bits hold
        if ctx % block:
            worst = torch.full((kv_heads, block - ctx % block, dim), 0x7F, dtype=torch.uint8)
            kc.view(torch.uint8)[table[b, ctx // block], :, ctx % block:] = worst
            vc.view(torch.uint8)[table[b, ctx // block], :, ctx % block:] = worst
    q = torch.randn(starts[-1] + 3, heads, dim, generator=g).bfloat16()  # three padding rows
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    out = torch.full_like(q, math.nan).to(device)
    o = kvc.cached_attention(q.to(device), *(t.to(device) for t in (kc, vc, ks, vs, table)), i32(context), i32(starts),
                             max(n for _, n in lens), max(context), out=out)
    assert o.data_ptr() == out.data_ptr() and (o[-3:] == 0).all()
    _check(o, want, size)
    # more new tokens than cached ones in all: the first see nothing
    context[0] = starts[1] - 2 if starts[1] > 2 else 0
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    o = kvc.cached_attention(q.to(device), *(t.to(device) for t in (kc, vc, ks, vs, table)), i32(context), i32(starts),
                             max(n for _, n in lens), max(context))
    assert (o[0] == 0).all()
    _check(o, want, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [6, 200])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_nan_value_reaches_the_rows_that_see_it_and_no_other(dim, new, device):
    g = torch.Generator().manual_seed(11)
    lens = [(30, new)]
    table, context, starts, blocks = _requests(lens, 32, g)
    kc, vc, ks, vs = _cache(blocks, 1, 32, dim, "fp8", g)
    at, d = 30 + new - 4, 5  # the value of the fourth last token
    vc.view(torch.uint8)[table[0, at // 32], 0, at % 32, d] = 0x7F
    q = torch.randn(new, 2, dim, generator=g).bfloat16()
    clean = vc.clone()
    clean.view(torch.uint8)[table[0, at // 32], 0, at % 32, d] = 0
    want, size = _attend_oracle(q, kc, clean, ks, vs, table, context, starts, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    o = kvc.cached_attention(q.to(device), *(t.to(device) for t in (kc, vc, ks, vs, table)), i32(context), i32(starts),
                             new, max(context)).cpu()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[new - 4:, :, d] = True
    assert torch.equal(o.isnan(), bad)
    _check(torch.where(bad, 0.0, o.double()), torch.where(bad, 0.0, want), size)


SPLITS = [  # [(cached, new)], heads, kv heads, head_dim, block: a request's keys over 16, 4, 2 and 1 blocks of threads
    ([(4000, 2), (9, 1)], 8, 2, 128, 64),
    ([(700, 1), (64, 1)] * 10, 4, 4, 64, 16),
    ([(500, 1), (0, 0), (1, 1)] * 15, 4, 4, 128, 32),
    ([(200, 1), (63, 1), (64, 1), (65, 1)] * 30, 4, 4, 128, 64),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("case", range(len(SPLITS)))
def test_attention_with_few_and_many_requests(case, fmt, device, monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], "SHAPES", SPLITS)
    test_attention_matches_64_bits(case, fmt, device)


@pytest.fixture
def no_bound(monkeypatch):
    """The host knows no useful bound of the lengths: all work in equal ranges."""
    attend = kvc.cached_attention

    def loose(*args, **kw):
        return attend(*args[:8], *(args[8:9] or (max(args[0].size(0), 1),)), 1 << 24, **kw)

    monkeypatch.setattr(kvc, "cached_attention", loose)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_without_a_bound(case, fmt, device, no_bound):
    test_attention_matches_64_bits(case, fmt, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[(70, 1), (3, 4)], [(40, 150), (0, 90)]])
def test_masks_and_nan_without_a_bound(lens, dim, device, no_bound):
    test_what_is_masked_does_not_count(dim, lens, "fp8", device)
    test_a_nan_value_reaches_the_rows_that_see_it_and_no_other(dim, 6 if lens[0][1] == 1 else 200, device)


@pytest.mark.parametrize("device", DEVICES)
def test_scales_far_apart_keep_the_small_values(device):
    """A block whose values are 2^24 times another's, and attention that looks at the small ones."""
    dim, block = 64, 16
    g = torch.Generator().manual_seed(5)
    table, context, starts, blocks = _requests([(31, 1)], block, g, spare=0)
    kc, vc, ks, vs = _cache(blocks, 1, block, dim, "int8", g)
    kc[:] = 0
    kc[table[0, 1].long(), 0, 3] = 100
    ks[:] = 1.0
    vs[table[0, 0].long()], vs[table[0, 1].long()] = 2.0 ** 12, 2.0 ** -12
    q = torch.full((1, 1, dim), 0.125).bfloat16()  # score 100 on key 19, 0 on the others
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    o = kvc.cached_attention(q.to(device), *(t.to(device) for t in (kc, vc, ks, vs, table)), i32(context), i32(starts), 1, 32)
    _check(o, want, size)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_takes_views(device):
    """Query rows of a packed projection, keys and values side by side, an output inside a larger one, another scale."""
    g = torch.Generator().manual_seed(9)
    lens, block, dim = [(50, 3), (9, 1)], 16, 64
    table, context, starts, blocks = _requests(lens, block, g)
    kc, vc, ks, vs = _cache(blocks, 2, block, dim, "int8", g)
    rows = torch.randn(4, 8, dim, generator=g).bfloat16()
    both, scales = torch.stack([kc, vc], 1).to(device), torch.stack([ks, vs], 1).to(device)
    out = torch.zeros(4, 6, dim, dtype=torch.bfloat16, device=device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    wide = torch.cat([table, table], 1).to(device)[:, : table.size(1)]
    kvc.cached_attention(rows.to(device)[:, :4], both[:, 0], both[:, 1], scales[:, 0], scales[:, 1], wide, i32(context),
                         i32(starts), 3, 53, scale=0.3, out=out[:, 1:5])
    want, size = _attend_oracle(rows[:, :4], kc, vc, ks, vs, table, context, starts, 0.3)
    _check(out[:, 1:5], want, size)
    assert (out[:, 0] == 0).all() and (out[:, 5] == 0).all()


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
@pytest.mark.parametrize("new", [1, 150])
def test_a_cache_beyond_32_bit_offsets(new):
    """Blocks whose bytes lie past 2^32: the write and the attention go there and nowhere else."""
    dim, heads, block = 128, 8, 64
    blocks = (1 << 32) // (heads * block * dim) + 40
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.empty(blocks, heads, block, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(blocks, heads, device="cuda") for _ in range(2))
    last = list(range(blocks - 10, blocks))
    table = torch.tensor([last], dtype=torch.int32, device="cuda")
    kc[:4], vc[:4] = 1, 2
    ctx = 200 + new
    k, v = (torch.randn(ctx, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = torch.tensor([last[j // block] * block + j % block for j in range(ctx)], dtype=torch.int32, device="cuda")
    kvc.append_kv(k, v, slots, kc, vc, ks, vs)
    q = torch.randn(new, 16, dim, generator=g, device="cuda").bfloat16()
    o = kvc.cached_attention(q, kc, vc, ks, vs, table, torch.tensor([ctx], dtype=torch.int32, device="cuda"),
                             torch.tensor([0, new], dtype=torch.int32, device="cuda"), new, ctx)
    near = torch.arange(10, dtype=torch.int32)[None]
    want, size = _attend_oracle(q, kc[-10:], vc[-10:], ks[-10:], vs[-10:], near, [ctx], [0, new], dim ** -0.5)
    _check(o, want, size)
    assert (kc[:4] == 1).all() and (vc[:4] == 2).all()


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_a_step_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(4)
    lens, block, dim = [(60, 1), (17, 1)], 16, 64
    table, context, starts, blocks = _requests(lens, block, g)
    kc, vc, ks, vs = (t.cuda() for t in _cache(blocks, 2, block, dim, "fp8", g))
    q = torch.randn(2, 4, dim, generator=g).bfloat16().cuda()
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    table, context, starts = table.cuda(), torch.tensor(context).int().cuda(), torch.tensor(starts).int().cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = kvc.cached_attention(q, kc, vc, ks, vs, table, context, starts, 1, 61)
    side.synchronize()
    _check(o, want, size)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = kvc.cached_attention(q, kc, vc, ks, vs, table, context, starts, 1, 61)
    q.copy_(q.flip(0).clone())
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    want, size = _attend_oracle(q, kc, vc, ks, vs, table.cpu(), context.tolist(), starts.tolist(), dim ** -0.5)
    _check(o, want, size)


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_do(device):
    kc = torch.zeros(2, 2, 16, 64, dtype=torch.int8, device=device)
    s = torch.ones(2, 2, device=device)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=device)
    ints = torch.zeros(0, dtype=torch.int32, device=device)
    kvc.append_kv(none, none, ints, kc, kc.clone(), s, s.clone())
    o = kvc.cached_attention(none, kc, kc, s, s, torch.full((1, 1), -1, dtype=torch.int32, device=device),
                             torch.zeros(1, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device))
    assert o.shape == (0, 2, 64)
    plan = kvc.plan_blocks(ints, ints, torch.tensor([2], dtype=torch.int32, device=device),
                           torch.zeros(0, 1, dtype=torch.int32, device=device), torch.arange(2, dtype=torch.int32, device=device), 16, 0)
    assert plan.query_start.tolist() == [0] and plan.state.tolist() == [2]


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_refusals():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(4, 2, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, ctx, start = i32([[0, 1]]), i32([5]), i32([0, 1])
    good = dict(q=q, k=kc, v=kc, ks=s, vs=s, table=table, ctx=ctx, start=start, mq=1, mc=5)

    def attend(**other):
        a = {**good, **other}
        return kvc.cached_attention(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["table"], a["ctx"], a["start"], a["mq"], a["mc"])

    attend()
    for other in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(k=kc.half()),
                  dict(k=kc.float(), v=kc.float()), dict(v=kc[:, :1]), dict(ks=s.double()), dict(ks=s[:3]),
                  dict(table=table.long()), dict(table=table[0]), dict(ctx=i32([5, 6])), dict(start=i32([0])),
                  dict(ctx=ctx.cpu()), dict(mq=0), dict(mc=0),
                  dict(k=kc[..., :48].contiguous(), v=kc[..., :48].contiguous()),
                  dict(k=torch.zeros(4, 2, 24, 64, dtype=torch.int8, device="cuda"),
                       v=torch.zeros(4, 2, 24, 64, dtype=torch.int8, device="cuda")),
                  dict(k=torch.zeros(4 * 2 * 16 * 64 + 8, dtype=torch.int8, device="cuda")[8:].view(4, 2, 16, 64))):
        with pytest.raises(RuntimeError):
            attend(**other)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in ((k[:, :1], k, i32([0, 1, 2])), (k, k[:2], i32([0, 1, 2])), (k, k, i32([0, 1])), (k.float(), k, i32([0, 1, 2])),
                (k, k, torch.zeros(3, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            kvc.append_kv(*bad, kc, kc.clone(), s, s.clone())
    with pytest.raises(RuntimeError):
        kvc.plan_blocks(i32([1]), i32([1, 2]), i32([4, 0]), table, i32([0]), 16, 1)
    with pytest.raises(RuntimeError):
        kvc.plan_blocks(i32([1]), i32([1]), i32([4, 0]), table, i32([0]), 24, 1)
    with pytest.raises(RuntimeError):
        kvc.plan_blocks(i32([1]), i32([1]), i32([4]), table, i32([0]), 16, 1)
