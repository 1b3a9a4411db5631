"""What one request asks for must not end the others (CPU forms)."""

import math

import pytest
import torch
from pydantic import ValidationError

from quantaweave_b200 import QuantaWeaveMoEForCausalLM, preset
from quantaweave_b200.inference.batching import BatchingWorker, ContinuousBatcher, GenerationRequest
from quantaweave_b200.inference.fast_decode import FastDecoder
from quantaweave_b200.tools.serve import GenerateRequest


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
