"""Penalties, biases and masks on logits against the definition in 64 bits. The kernel computes in 32 bits (a handful of
roundings, 2^-24 each, of numbers no larger than the sums of magnitudes here) and rounds once to the logits' type: 2^-24,
2^-11 or 2^-8 of the result, doubled, plus 2^-21 of the terms' magnitudes."""

import math

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200.ops.logits import pack_mask, process_logits

DEVICES = ["cpu", pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")])]
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def _oracle(x, history, used, prompt, rep, freq, pres, bias, bias_rows, allowed, mask_rows):
    x = x.double()
    size = x.abs()
    out = x.clone()
    for r in range(x.size(0)):
        for id_ in set(history[r, : used[r]].tolist()):
            if not 0 <= id_ < x.size(1):
                continue
            y = out[r, id_] / rep[r] if out[r, id_] > 0 else out[r, id_] * rep[r]
            size[r, id_] += y.abs()
            made = history[r, prompt[r]: used[r]].tolist().count(id_)
            if made:
                y = y - made * freq[r] - pres[r]
                size[r, id_] += made * abs(freq[r]) + abs(pres[r])
            out[r, id_] = y
        if bias is not None and 0 <= bias_rows[r] < bias.size(0):
            out[r] += bias[bias_rows[r]].double()
            size[r] += bias[bias_rows[r]].double().abs()
        if allowed is not None and 0 <= mask_rows[r] < allowed.size(0):
            out[r] = torch.where(allowed[mask_rows[r]], out[r], -math.inf)
    return out, size


def _check(got, want, size, dtype):
    got = got.cpu().double()
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]) and torch.equal(got.isnan(), want.isnan())
    over = (got - want).abs()[fine] - (EPS[dtype] * want.abs() + 2.0 ** -21 * size)[fine]
    assert not over.numel() or over.max() <= 0, over.max().item()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,length", [(1, 1, 1), (1, 31, 5), (3, 1000, 40), (2, 1027, 200), (5, 8193, 17), (2, 20011, 300),
                                               (70, 515, 9)])
def test_logits_match_64_bits(rows, vocab, length, dtype, device):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (4 * torch.randn(rows, vocab + 5, generator=g)).to(dtype)
    x[0, 0] = -math.inf
    history = torch.randint(-2, min(vocab + 3, 60), (rows, length + 2), generator=g).int()  # some ids are no ids
    history[:, -1] = vocab - 1
    used = torch.randint(0, length + 3, (rows,), generator=g).int()
    prompt = (used * torch.rand(rows, generator=g)).int()
    rep = 1 + torch.rand(rows, generator=g)
    freq, pres = torch.randn(rows, generator=g), torch.rand(rows, generator=g)
    bias = torch.randn(3, vocab, generator=g)
    bias_rows = (torch.arange(rows) % 5 - 1).int()  # none, a row, and one that there is not
    allowed = torch.rand(2, vocab, generator=g) < 0.5
    mask_rows = (torch.arange(rows) % 4 - 1).int()
    d = lambda t: t.to(device)  # noqa: E731
    padded = d(x)[:, :vocab]  # rows on odd boundaries
    kw = dict(history=d(history), history_lens=d(used), prompt_lens=d(prompt), repetition=d(rep), frequency=d(freq),
              presence=d(pres), bias=d(bias), bias_rows=d(bias_rows), mask=d(pack_mask(allowed)), mask_rows=d(mask_rows))
    want, size = _oracle(x[:, :vocab], history, used, prompt, rep, freq, pres, bias, bias_rows, allowed, mask_rows)
    _check(process_logits(padded, **kw), want, size, dtype)
    own = padded.clone(memory_format=torch.contiguous_format)
    assert process_logits(own, out=own, **kw).data_ptr() == own.data_ptr()  # in place
    _check(own, want, size, dtype)
    inside = torch.zeros(rows, vocab + 3, dtype=dtype, device=device)
    process_logits(padded, out=inside[:, 1:vocab + 1], **kw)  # the output's boundaries are not the input's
    _check(inside[:, 1:vocab + 1], want, size, dtype)
    assert (inside[:, 0] == 0).all() and (inside[:, vocab + 1:] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_each_part_alone(device):
    g = torch.Generator().manual_seed(0)
    rows, vocab = 2, 77
    x = torch.randn(rows, vocab, generator=g)
    x[1, 3] = math.nan
    history = torch.tensor([[5, 5, 9, 3], [3, 0, 0, 0]]).int()
    used, prompt = torch.tensor([4, 2]).int(), torch.tensor([1, 1]).int()
    one, zero = torch.ones(rows), torch.zeros(rows)
    bias, allowed = torch.randn(rows, vocab, generator=g), torch.rand(rows, vocab, generator=g) < 0.3
    d = lambda t: t.to(device)  # noqa: E731
    own = torch.arange(rows)
    past = dict(history=d(history), history_lens=d(used), prompt_lens=d(prompt))
    for kw, args in ((dict(), (one, zero, zero, None, None)),
                     (dict(**past, repetition=d(one * 1.7)), (one * 1.7, zero, zero, None, None)),
                     (dict(**past, frequency=d(one * 0.3)), (one, one * 0.3, zero, None, None)),
                     (dict(**past, presence=d(one * 0.4)), (one, zero, one * 0.4, None, None)),
                     (past, (one, zero, zero, None, None)),
                     (dict(bias=d(bias)), (one, zero, zero, bias, None)),
                     (dict(mask=d(pack_mask(allowed))), (one, zero, zero, None, allowed))):
        rep, freq, pres, b, a = args
        want, size = _oracle(x, history, used, prompt, rep, freq, pres, b, own, a, own)
        _check(process_logits(d(x), **kw), want, size, torch.float32)


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_logits_refusals():
    x = torch.zeros(2, 64, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for kw in (dict(history=i32([[1], [2]])), dict(repetition=torch.ones(2, device="cuda")),
               dict(history=i32([[1], [2]]), history_lens=i32([1])), dict(history=i32([[1]]), history_lens=i32([1, 1])),
               dict(bias=torch.zeros(3, 64, device="cuda")), dict(bias=torch.zeros(2, 63, device="cuda")),
               dict(bias=torch.zeros(2, 64)), dict(mask=i32([[1], [2]])), dict(mask=torch.zeros(2, 2, device="cuda")),
               dict(mask=i32([[1, 2]])), dict(out=torch.zeros(2, 64, device="cuda").half())):
        with pytest.raises(RuntimeError):
            process_logits(x, **kw)
    with pytest.raises(RuntimeError):
        process_logits(x.double())
    with pytest.raises(RuntimeError):
        process_logits(x.T)
    assert process_logits(x[:0]).shape == (0, 64)
