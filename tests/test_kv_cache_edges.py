"""The block-wise 8-bit KV cache at its edges: held scales that are none, numbers far below their row's largest, no heads,
offsets that do not fit, inputs that ask for gradients."""

import math

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200.ops import kv_cache as kvc
from quantaweave_b200.ops.logits import process_logits

GPU = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")]
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("held", [0.0, math.nan, math.inf])
def test_a_held_scale_that_is_none_sets_no_scale(held, fmt, device):
    """A cache that was never written holds zeros, its scales as well: a write into the middle of a block takes the new
    numbers' own scale."""
    x = torch.tensor([0.75, -0.5]).repeat(16)[None, None].bfloat16()
    kc, vc = (torch.zeros(1, 1, 16, 32, dtype=kvc.FORMATS[fmt], device=device) for _ in range(2))
    ks, vs = (torch.full((1, 1), held, device=device) for _ in range(2))
    kvc.append_kv(x.to(device), x.to(device), torch.tensor([5], dtype=torch.int32, device=device), kc, vc, ks, vs)
    scale = 2.0 ** (-9 if fmt == "fp8" else -7)  # 0.75 = 384 * 2^-9 = 96 * 2^-7
    for codes, scales in ((kc, ks), (vc, vs)):
        assert scales.tolist() == [[scale]]
        assert torch.equal(codes[0, 0, 5].cpu().double() * scale, x[0, 0].double())


@pytest.mark.parametrize("device", DEVICES)
def test_inputs_that_ask_for_gradients_are_refused(device):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    kc = torch.zeros(2, 2, 16, 32, dtype=torch.int8, device=device)
    s = torch.ones(2, 2, device=device)
    x = torch.zeros(1, 2, 32, dtype=torch.bfloat16, device=device, requires_grad=True)
    logits = torch.zeros(1, 40, device=device)
    ones, bias = (torch.ones(shape, device=device, requires_grad=True) for shape in ((1,), (1, 40)))
    calls = (lambda: kvc.cached_attention(x, kc, kc, s, s, i32([[0]]), i32([1]), i32([0, 1])),
             lambda: kvc.append_kv(x, x.detach(), i32([3]), kc, kc.clone(), s, s.clone()),
             lambda: kvc.append_kv(x.detach(), x, i32([3]), kc, kc.clone(), s, s.clone()),
             lambda: process_logits(logits.clone().requires_grad_()), lambda: process_logits(logits, bias=bias),
             lambda: process_logits(logits, history=i32([[1]]), history_lens=i32([1]), repetition=ones))
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens", [0, 3])
def test_no_query_heads_give_an_empty_output(tokens, device):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    kc = torch.zeros(2, 2, 16, 64, dtype=torch.int8, device=device)
    s = torch.ones(2, 2, device=device)
    q = torch.zeros(tokens, 0, 64, dtype=torch.bfloat16, device=device)
    assert kvc.cached_attention(q, kc, kc, s, s, i32([[0]]), i32([5]), i32([0, tokens])).shape == (tokens, 0, 64)


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_a_cache_without_heads_is_refused():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kc = torch.zeros(2, 0, 16, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(2, 0, device="cuda")
    x = torch.zeros(3, 0, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="head"):
        kvc.append_kv(x, x, i32([0, 1, 2]), kc, kc.clone(), s, s.clone())
    with pytest.raises(RuntimeError, match="head"):
        kvc.cached_attention(x, kc, kc, s, s, i32([[0]]), i32([5]), i32([0, 3]))


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("starts,over", [([0, 1000] * 4, True), ([0, 1000, 990, 1000, 1, 1000], True), ([0, 500, 700, 300], False),
                                         ([7, 1000, -9], False), ([0, 1000, 1400], False)])
def test_row_offsets_that_do_not_ascend_stay_inside_the_buffers(starts, over, dim):
    """Overlapping requests have more row tiles than the rows of q allow: the prompt kernel leaves the surplus out and sets the
    status word, the rest of the output is that of some request; the next call is as ever."""
    from quantaweave_b200.ops import ext

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    requests, tokens = len(starts) - 1, 1000
    kc = torch.ones(64, 1, 16, dim, dtype=torch.int8, device="cuda")
    s = torch.ones(64, 1, device="cuda")
    table = torch.arange(64, device="cuda", dtype=torch.int32).expand(requests, 64).contiguous()
    q = torch.randn(tokens, 1, dim, generator=torch.Generator("cuda").manual_seed(0), device="cuda").bfloat16()
    out = torch.zeros_like(q)
    kvc.cached_attention(q, kc, kc, s, s, table, i32([1000] * requests), i32(starts), tokens, 1024, out=out)
    assert (ext().read_status(True) != 0) == over
    assert ((out == 1) | (out == 0)).all()  # every value is 1
    o = kvc.cached_attention(q, kc, kc, s, s, table[:1], i32([1000]), i32([0, tokens]), tokens, 1024)
    assert (o == 1).all() and ext().read_status(True) == 0


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_a_table_of_more_tokens_than_32_bits_is_refused():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    block = 1 << 20
    kc = torch.zeros(1, 1, block, 32, dtype=torch.int8, device="cuda")
    s = torch.ones(1, 1, device="cuda")
    q = torch.zeros(1, 1, 32, dtype=torch.bfloat16, device="cuda")
    for width, fits in ((2047, True), (2048, False), (4096, False)):
        table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
        if fits:
            kvc.cached_attention(q, kc, kc, s, s, table, i32([3]), i32([0, 1]), 1, 3)
        else:
            with pytest.raises(RuntimeError, match="tokens"):
                kvc.cached_attention(q, kc, kc, s, s, table, i32([3]), i32([0, 1]), 1, 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("new", [1, 6, 200])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_query_numbers_far_below_their_rows_largest_count(dim, new, fmt, device):
    """A query row whose largest number meets keys of zero, and two numbers 2^-20 of it, unlike in their last bit, that meet large
    keys of opposite sign: the score is that last bit. The tolerance is that of the other attention tests."""
    from test_kv_cache import _attend_oracle, _check, _requests

    g = torch.Generator().manual_seed(dim + new)
    table, context, starts, blocks = _requests([(40, new)], 16, g)
    codes = torch.zeros(blocks, 2, 16, dim)
    codes[..., 1] = 120 * (torch.rand(blocks, 2, 16, generator=g) < 0.3)
    codes[..., 2] = -codes[..., 1]
    kc = codes.to(kvc.FORMATS[fmt])
    vc = torch.randint(-100, 101, codes.shape, generator=g).float().to(kvc.FORMATS[fmt])
    ks, vs = torch.full((blocks, 2), 2.0 ** 19 * math.sqrt(dim / 64)), torch.full((blocks, 2), 2.0 ** -6)
    q = torch.zeros(new, 4, dim)
    q[..., 0], q[..., 1], q[..., 2] = 64.0, 64 * 2.0 ** -20 * 255 / 128, 64 * 2.0 ** -20 * 254 / 128
    q = q.bfloat16()
    want, size = _attend_oracle(q, kc, vc, ks, vs, table, context, starts, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    o = kvc.cached_attention(*(t.to(device) for t in (q, kc, vc, ks, vs, table)), i32(context), i32(starts), new, context[0])
    _check(o, want, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 200])
def test_query_rows_at_the_ends_of_bf16(new, device):
    """Rows whose largest number is the largest of bf16, and rows of the smallest normal one, with a scale that makes their scores
    ordinary."""
    from test_kv_cache import _attend_oracle, _check, _requests

    g = torch.Generator().manual_seed(new)
    table, context, starts, blocks = _requests([(40, new)], 16, g)
    kc = torch.randint(-127, 128, (blocks, 2, 16, 64), generator=g).to(torch.int8)
    vc = torch.randint(-127, 128, (blocks, 2, 16, 64), generator=g).to(torch.int8)
    vs = torch.full((blocks, 2), 2.0 ** -6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    for top, unit in ((torch.finfo(torch.bfloat16).max, 2.0 ** -120), (2.0 ** -100, 2.0 ** 108)):
        q = (torch.rand(new, 4, 64, generator=g) * 2 - 1) * top
        q[..., 3] = top
        q = q.bfloat16()
        ks = torch.full((blocks, 2), unit * 2.0 ** -17)
        args = (q, kc, vc, ks, vs, table)
        want, size = _attend_oracle(*args, context, starts, 0.125)
        _check(kvc.cached_attention(*(t.to(device) for t in args), i32(context), i32(starts), new, context[0], 0.125), want, size)
