"""What one request asks for must not end the others (CPU forms)."""

import asyncio
import math

import pytest
import torch
from pydantic import ValidationError
from test_tools_cpu import _train

from quantaweave_b200 import QuantaWeaveMoEForCausalLM, preset
from quantaweave_b200.inference.batching import BatchingWorker, ContinuousBatcher, GenerationRequest
from quantaweave_b200.inference.fast_decode import FastDecoder
from quantaweave_b200.tools.serve import GenerateRequest, Server, main


def _batcher(cache="int8", rows=3):
    torch.manual_seed(0)
    model = QuantaWeaveMoEForCausalLM(preset("tiny-cpu", max_sequence_length=65)).eval()
    kw = {} if cache == "dense" else {"cache_block": 16}
    return ContinuousBatcher(FastDecoder(model, torch.device("cpu"), max_batch=rows, kv_cache=cache, **kw))


@pytest.mark.parametrize("bad", [dict(frequency_penalty=-1e39), dict(frequency_penalty=math.nan), dict(presence_penalty=math.inf),
                                 dict(presence_penalty=math.nan), dict(repetition_penalty=1e-40), dict(repetition_penalty=math.nan),
                                 dict(repetition_penalty=math.inf), dict(repetition_penalty=-1.0)])
def test_penalties_beyond_32_bit_logits_are_refused(bad):
    with pytest.raises(ValidationError):
        GenerateRequest(prompt="the", **bad)
    batcher = _batcher()
    with pytest.raises(ValueError, match="penalty"):
        batcher.submit(GenerationRequest([1, 2], 4, **bad))
    assert batcher.pending() == 0
    worker = BatchingWorker(batcher)
    try:
        neighbour = worker.submit(GenerationRequest([3, 4], 12, temperature=1.0))
        with pytest.raises(ValueError, match="penalty"):
            worker.submit(GenerationRequest([1, 2], 4, temperature=1.0, **bad))
        assert len(neighbour.wait(30)) == 12 and neighbour.finish_reason == "length" and worker.error is None
    finally:
        worker.close()


@pytest.mark.parametrize("edge", [dict(frequency_penalty=-1e6), dict(presence_penalty=1e6), dict(repetition_penalty=1e-6),
                                  dict(repetition_penalty=1e6)])
def test_penalties_at_their_limits_can_be_sampled(edge):
    batcher = _batcher()
    request = batcher.submit(GenerationRequest([1, 2, 3], 20, temperature=0.7, **edge))
    batcher.run_until_idle()
    assert len(request.tokens) == 20


def _raises(made):
    raise RuntimeError("no such state")


VOCAB = 512  # of the tiny preset


@pytest.mark.parametrize("cache", ["dense", "int8"])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("bad", [dict(allowed=_raises), dict(allowed=lambda made: torch.zeros(VOCAB, dtype=torch.bool)),
                                 dict(allowed=lambda made: torch.ones(VOCAB - 1, dtype=torch.bool)),
                                 dict(allowed=lambda made: None if len(made) == 2 else torch.ones(VOCAB, dtype=torch.bool)),
                                 dict(logit_bias=torch.full((VOCAB,), -math.inf)), dict(logit_bias=torch.zeros(3))])
def test_a_request_that_cannot_be_sampled_ends_alone(bad, temperature, cache):
    alone = _batcher(cache)
    want = [alone.submit(GenerationRequest([5, 6], 9, temperature=1.0, seed=3)), alone.submit(GenerationRequest([7], 11))]
    alone.run_until_idle()
    worker = BatchingWorker(_batcher(cache))
    try:
        beside = [worker.submit(GenerationRequest([5, 6], 9, temperature=1.0, seed=3)), None]
        broken = worker.submit(GenerationRequest([1, 2, 3], 9, temperature=temperature, **bad))
        beside[1] = worker.submit(GenerationRequest([7], 11))
        for w, b in zip(want, beside):
            assert b.wait(30) == w.tokens and b.finish_reason == "length"
        broken.wait(30)
        assert broken.finish_reason.startswith("error: ") and len(broken.tokens) in (0, 2)
        assert worker.error is None and worker.batcher.pending() == 0
        cache_state = worker.batcher.decoder.cache
        assert cache_state is None or cache_state.state.tolist() == [cache_state.blocks, 0, 0, 0]
    finally:
        worker.close()


@pytest.mark.parametrize("given", [list, torch.Tensor.int, lambda m: m.numpy()])
def test_a_grammar_may_give_its_mask_in_other_forms(given):
    even = torch.arange(VOCAB) % 2 == 0
    batcher = _batcher()
    request = batcher.submit(GenerationRequest([1, 2, 3], 8, allowed=lambda made: given(even)))
    batcher.run_until_idle()
    assert len(request.tokens) == 8 and all(t % 2 == 0 for t in request.tokens)


@pytest.mark.parametrize("options", [dict(kv_cache="fp8"), dict(cache_blocks=8), dict(batching=2, cache_blocks=8)])
def test_cache_options_that_would_be_ignored_are_refused(options, tmp_path, capsys):
    with pytest.raises(ValueError, match="batching|kv-cache"):
        Server(tmp_path / "none", None, torch.device("cpu"), "fp32", **options)
    flags = [f"--{name.replace('_', '-')}={value}" for name, value in options.items()]
    with pytest.raises(SystemExit):
        main(["--checkpoint", str(tmp_path / "none"), "--device", "cpu", *flags])
    assert "needs" in capsys.readouterr().err


def test_a_server_whose_pool_is_smaller_than_a_context_shortens_the_request(tmp_path):
    _train(tmp_path, steps=1, sequence_length=160)
    server = Server(tmp_path / "out", None, torch.device("cpu"), "fp32", batching=2, kv_cache="fp8", cache_blocks=1)
    try:
        long = asyncio.run(server.generate(GenerateRequest(prompt="the cat " * 10, tokens=40, temperature=0.0, stop=[])))
        assert long["truncated_context"] and 1 <= long["tokens"] <= 40
        many = asyncio.run(server.generate(GenerateRequest(prompt="the", tokens=150, temperature=0.0, stop=[])))
        assert 1 <= many["tokens"] <= 63 and server.worker.error is None
    finally:
        server.close()
