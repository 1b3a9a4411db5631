"""A pool of cache blocks smaller than every row's full context: who gets blocks, and what happens when they run out."""

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200 import QuantaWeaveMoEForCausalLM, preset
from quantaweave_b200.inference.batching import ContinuousBatcher, GenerationRequest
from quantaweave_b200.inference.fast_decode import FastDecoder
from quantaweave_b200.inference.paged_cache import PoolExhausted
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


@pytest.mark.parametrize("device", DEVICES)
def test_each_use_of_a_decoder_begins_with_the_whole_pool(device):
    """Blocks left by a batcher, by more rows, or by a generation before: none is missing afterwards."""
    model = _model(device)
    prompt = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(0))
    want = _decoder(model, device, 4).generate(prompt, 40)

    def batcher_first(dec):
        batcher = ContinuousBatcher(dec)
        for _ in range(4):
            batcher.submit(GenerationRequest(list(range(1, 12)), 20))
        batcher.run_until_idle()
        assert dec.cache.state.tolist() == [8, 0, 0, 0, 0]

    def wide_first(dec):
        dec.generate(torch.arange(40).view(2, 20), 41)

    for before in (batcher_first, wide_first):
        dec = _decoder(model, device, 4, blocks=8)
        before(dec)
        got = dec.generate(prompt, 40)  # 99 tokens are kept: seven of the eight blocks
        assert dec.cache.state.tolist() == [1, 7, 0, 0, 0]
        assert device == "cuda" or torch.equal(got, want)
        again = ContinuousBatcher(dec)
        request = again.submit(GenerationRequest(prompt[0].tolist(), 40))
        again.run_until_idle()
        assert request.finish_reason == "length" and dec.cache.state.tolist() == [8, 0, 0, 0, 0]
        assert device == "cuda" or request.tokens == want[0].tolist()


@pytest.mark.parametrize("device", DEVICES)
def test_a_pool_that_is_too_small_is_an_error(device):
    model = _model(device)
    dec = _decoder(model, device, 2, blocks=3)
    prompts = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(1))
    whole = _decoder(model, device, 2)
    with pytest.raises(PoolExhausted, match="4 cache blocks, the pool has 3"):
        dec.generate(prompts, 10)
    assert dec.cache.state.tolist() == [3, 0, 0]  # refused before any work
    got = dec.generate(prompts[:1], 29)           # 48 tokens are kept
    assert device == "cuda" or torch.equal(got, whole.generate(prompts[:1], 29))
    with pytest.raises(PoolExhausted):
        dec.generate(prompts[:1], 30)
    with pytest.raises(PoolExhausted):
        dec.feed(list(range(49)))
    dec.feed(list(range(47)))
    dec.append(1)
    length = dec.length
    for _ in range(2):
        with pytest.raises(PoolExhausted, match="a context of 49 tokens"):
            dec.append(2)
    assert dec.length == length == 48 and dec.cache.state.tolist() == [0, 3, 0]
    dec.feed([1, 2])  # begins anew
    assert dec.cache.state.tolist() == [2, 1, 0]
    with pytest.raises(PoolExhausted):
        list(dec.stream(list(range(40)), 20, temperature=0.0))


@pytest.mark.parametrize("device", DEVICES)
def test_steps_and_prompts_without_room_are_refused(device):
    model = _model(device)
    dec = _decoder(model, device, 2, blocks=3)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(2))
    with pytest.raises(PoolExhausted):
        dec._prefill(ids)
    dec._prefill(ids[:, :16])
    at = lambda *x: torch.tensor(x, device=device)  # noqa: E731
    with pytest.raises(PoolExhausted):
        dec.run_step(ids[:, 16].to(device), at(16, 16))
    assert dec.cache.state.tolist() == [1, 1, 1]
    dec.run_step(ids[:, 15].to(device), at(15, 15))                       # again the last token: no block
    dec.run_step(at(7, 0), at(0, 16), at(0, 1))                           # one request alone
    assert dec.cache.state.tolist() == [0, 1, 2]
    with pytest.raises(PoolExhausted):
        dec.run_step(at(7, 0), at(16, 0), at(1, 0))
    with pytest.raises(PoolExhausted):
        dec._prefill(ids[:1, :33], first_row=0)                           # the other row holds two of the three
    with pytest.raises(PoolExhausted, match="at most 8"):
        _decoder(model, device, 1)._prefill(torch.zeros(1, 129, dtype=torch.long))


@pytest.mark.parametrize("precision", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", [dict(), dict(norm_type="layernorm", position_embedding="learned", attention_bias=True)])
def test_cpu_decoding_in_every_precision(layout, precision):
    cfg = preset("tiny-cpu", max_sequence_length=65, **layout)
    torch.manual_seed(0)
    model = QuantaWeaveMoEForCausalLM(cfg).eval()
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(3))
    logits = []
    for cache in ("dense", "int8"):
        dec = FastDecoder(model, torch.device("cpu"), precision, max_batch=2, kv_cache=cache)
        dec._prefill(ids[:, :-1])
        logits.append(dec.run_step(ids[:, -1], torch.full((2,), 19)).clone())
    assert (logits[0] - logits[1]).abs().max() < 0.05 * logits[0].abs().max() + 0.05  # the 8-bit cache's own tolerance
