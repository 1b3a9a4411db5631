"""Each step of the logits' processing is one 32-bit operation: a division is a division."""

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200.ops.logits import process_logits

DEVICES = ["cpu", pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")])]


@pytest.mark.parametrize("device", DEVICES)
def test_repetition_is_a_correctly_rounded_division(device):
    g = torch.Generator().manual_seed(0)
    rows, vocab = 8, 4099
    x = 5 * torch.randn(rows, vocab, generator=g)
    rep = torch.tensor([1.3, 1.1, 0.7, 1.0, 3.0, 1e-6, 1e6, 2.0 ** 126 * 1.3])
    history = torch.arange(vocab, dtype=torch.int32).expand(rows, vocab).contiguous()
    used = torch.full((rows,), vocab, dtype=torch.int32)
    got = process_logits(x.to(device), history=history.to(device), history_lens=used.to(device), prompt_lens=used.to(device),
                         repetition=rep.to(device))
    want = torch.where(x > 0, x.double() / rep.double()[:, None], x.double() * rep.double()[:, None]).float()
    assert torch.equal(got.cpu(), want)
