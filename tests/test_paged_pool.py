"""A pool of cache blocks smaller than every row's full context: who gets blocks, and what happens when they run out."""

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200 import QuantaWeaveMoEForCausalLM, preset
from quantaweave_b200.inference.batching import ContinuousBatcher, GenerationRequest
from quantaweave_b200.inference.fast_decode import FastDecoder
from quantaweave_b200.ops import kv_cache as kvc

GPU = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")]
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


def _model(device):
    cfg = preset("tiny-cpu", max_sequence_length=129, hidden_size=256, attention_heads=4, ffn_size=256)
    torch.manual_seed(0)
    return QuantaWeaveMoEForCausalLM(cfg).eval().to(device)


def _decoder(model, device, rows, blocks=None):
    return FastDecoder(model, torch.device(device), max_batch=rows, kv_cache="int8", cache_block=16, cache_blocks=blocks)


@pytest.mark.parametrize("device", DEVICES)
def test_a_request_without_new_tokens_takes_no_blocks(device):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table, free = torch.full((3, 4), -1, dtype=torch.int32, device=device), i32([3, 1, 2, 0])
    plan = kvc.plan_blocks(i32([40, 5, 200]), i32([0, 2, 0]), i32([4, 0, 0, 0]), table, free, 16, 2)
    assert plan.state.tolist() == [3, 0, 1, 0] and plan.missing.tolist() == [0]
    assert table.tolist() == [[-1] * 4, [0, -1, -1, -1], [-1] * 4]
    assert plan.slot_map.tolist() == [5, 6] and plan.query_start.tolist() == [0, 0, 2, 2]


@pytest.mark.parametrize("device", DEVICES)
def test_rows_left_out_of_a_step_take_no_blocks(device):
    model = _model(device)
    want = _decoder(model, device, 1).generate(torch.arange(1, 35)[None], 30)
    dec = _decoder(model, device, 2, blocks=6)
    dec.generate(torch.arange(40).view(2, 20), 20)  # positions up to 38 in both rows
    dec.cache.release_rows([0, 1])
    logits = dec.feed(list(range(1, 35)))
    got = []
    for _ in range(30):  # 64 tokens: four of the six blocks
        got.append(int(logits.argmax()))
        logits = dec.append(got[-1])
    assert dec.cache.state.tolist() == [2, 4, 0]
    if device == "cpu":
        assert got == want[0].tolist()
