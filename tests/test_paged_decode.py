"""Decoding and continuous batching through the block-wise 8-bit KV cache."""

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200 import QuantaWeaveConfig, QuantaWeaveMoEForCausalLM, preset
from quantaweave_b200.inference.batching import ContinuousBatcher, GenerationRequest
from quantaweave_b200.inference.fast_decode import FastDecoder, Unsupported
from quantaweave_b200.inference.paged_cache import PagedKVCache

CPU = torch.device("cpu")
GPU = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")]
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


def _model(**kw):
    cfg = preset("tiny-cpu", **{"max_sequence_length": 129, "hidden_size": 256, "attention_heads": 4, "ffn_size": 256, **kw})
    torch.manual_seed(0)
    model = QuantaWeaveMoEForCausalLM(cfg).eval()
    for moe in model.moes():
        moe.drop_overflow_tokens = False
    return model


def _close(got, want):
    # 8-bit keys and values move the logits by a few percent of their range (an int8 number is off by up to 2^-7 of its
    # block's largest, an fp8 one by 2^-4 of itself); the native decoder's own tolerance is the same
    return (got.float().cpu() - want.float().cpu()).abs().max() < 0.05 * want.abs().max() + 0.05


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("layout", [dict(), dict(norm_type="layernorm", position_embedding="learned", attention_bias=True,
                                                 kv_heads=2)])
def test_paged_decoding_stays_close_to_the_dense_cache(layout, fmt):
    model = _model(**layout)
    prompts = torch.randint(0, 512, (3, 40), generator=torch.Generator().manual_seed(1))
    dense = FastDecoder(model, CPU, max_batch=3)
    paged = FastDecoder(model, CPU, max_batch=3, kv_cache=fmt, cache_block=16)
    assert "block-wise" in paged.description
    for dec in (dense, paged):
        dec._prefill(prompts[:, :30])
    for i in range(30, 40):
        pos = torch.full((3,), i)
        assert _close(paged.run_step(prompts[:, i], pos), dense.run_step(prompts[:, i], pos)), i
    assert paged.generate(prompts, 6).shape == (3, 6)


def test_prompts_read_in_pieces_of_whole_blocks_leave_the_same_cache():
    model = _model()
    ids = torch.randint(0, 512, (2, 70), generator=torch.Generator().manual_seed(2))
    whole = FastDecoder(model, CPU, max_batch=2, kv_cache="fp8", cache_block=16)
    pieces = FastDecoder(model, CPU, max_batch=2, kv_cache="fp8", cache_block=16, prefill_chunk=32)
    out = []
    for dec in (whole, pieces):
        dec._prefill(ids[:, :-1])
        out.append(dec.run_step(ids[:, -1], torch.full((2,), 69)).clone())
    assert torch.allclose(*out, atol=1e-3)


def test_the_single_request_interface_survives_a_full_context():
    model = _model(max_sequence_length=41)
    dec = FastDecoder(model, CPU, kv_cache="int8", cache_block=16)
    dec.feed([1, 2, 3])
    for t in range(60):  # the context fills twice: the oldest half is dropped and the rest read again
        dec.append(t)
    assert 0 < dec.length <= dec.capacity and int(dec.cache.state[0]) == dec.cache.blocks - int(dec.cache.state[1])
    assert len(list(dec.stream([4, 5], 7, temperature=0.0))) == 7


PROMPTS = [[1, 2, 3], list(range(5, 40)), [7, 8, 9, 10, 11], [2, 2], [3, 1, 4, 1, 5, 9] * 5, [6]]
BUDGETS = [20, 7, 30, 6, 18, 40]


@pytest.mark.parametrize("device", DEVICES)
def test_a_small_pool_is_shared_and_comes_back(device):
    model = _model().to(device)
    blocks = 8  # six slots of 128 tokens would need 48 blocks of 16
    dec = FastDecoder(model, torch.device(device), max_batch=4, kv_cache="fp8", cache_block=16, cache_blocks=blocks)
    assert dec.uses_graph == (device == "cuda")
    batcher = ContinuousBatcher(dec)
    requests = [batcher.submit(GenerationRequest(p, n)) for p, n in zip(PROMPTS, BUDGETS)]
    most = 0
    while batcher.pending():
        batcher.step()
        most = max(most, blocks - int(dec.cache.state[0]))
    assert [len(r.tokens) for r in requests] == BUDGETS and all(r.finish_reason == "length" for r in requests)
    assert 4 <= most <= blocks
    assert int(dec.cache.state[0]) == blocks and (dec.cache.state[1:] == 0).all() and (dec.cache.block_table == -1).all()
    assert sorted(dec.cache.free_blocks.tolist()) == list(range(blocks))  # none lost, none doubled
    if device == "cpu":  # a request's tokens do not depend on its company
        for p, n, r in zip(PROMPTS, BUDGETS, requests):
            alone = ContinuousBatcher(FastDecoder(model, CPU, max_batch=4, kv_cache="fp8", cache_block=16))
            again = alone.submit(GenerationRequest(p, n))
            alone.run_until_idle()
            assert again.tokens == r.tokens
    small = ContinuousBatcher(FastDecoder(model, torch.device(device), kv_cache="fp8", cache_block=16, cache_blocks=4))
    with pytest.raises(ValueError, match="cache blocks"):
        small.submit(GenerationRequest(list(range(60)), 20))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache", ["dense", "int8"])
def test_penalties_and_grammar_masks_shape_what_is_generated(cache, device):
    model = _model().to(device)
    vocab = model.config.vocab_size
    even = torch.arange(vocab) % 2 == 0

    def run(*requests):
        batcher = ContinuousBatcher(FastDecoder(model, torch.device(device), max_batch=3, kv_cache=cache))
        for r in requests:
            batcher.submit(r)
        batcher.run_until_idle()
        return [r.tokens for r in requests]

    plain = run(GenerationRequest([1, 2, 3], 24))[0]
    fresh, masked, beside = run(GenerationRequest([1, 2, 3], 24, presence_penalty=1e4),
                                GenerationRequest([1, 2, 3], 24, allowed=lambda made: even),
                                GenerationRequest([1, 2, 3], 24))
    assert len(set(fresh)) == 24                     # no generated id twice
    assert all(t % 2 == 0 for t in masked)
    if device == "cpu":
        assert beside == plain                       # the others are left alone
    # a grammar may look at what was generated: alternately even and odd
    turns = run(GenerationRequest([9], 12, allowed=lambda made: even if len(made) % 2 == 0 else ~even))[0]
    assert [t % 2 for t in turns] == [0, 1] * 6
    with pytest.raises(ValueError, match="repetition_penalty"):
        run(GenerationRequest([1], 2, repetition_penalty=0.0))


def test_a_failed_request_gives_its_blocks_back(monkeypatch):
    dec = FastDecoder(_model(), CPU, max_batch=2, kv_cache="fp8", cache_block=16, cache_blocks=4)
    batcher = ContinuousBatcher(dec)
    original = dec._prefill

    def prefill(prompts, first_row=0):
        original(prompts, first_row)
        if prompts[0, 0] == 63:
            raise RuntimeError("bad prompt")

    monkeypatch.setattr(dec, "_prefill", prefill)
    bad = batcher.submit(GenerationRequest([63] * 40, 8))
    with pytest.raises(RuntimeError, match="bad prompt"):
        batcher.step()
    assert bad.finish_reason.startswith("error")
    good = batcher.submit(GenerationRequest([1] * 50, 10))  # needs all four blocks
    batcher.run_until_idle()
    assert len(good.tokens) == 10 and int(dec.cache.state[0]) == 4


def test_refusals():
    model = _model()
    for kw in (dict(kv_cache="int4"), dict(kv_cache="fp8", cache_block=24), dict(kv_cache="fp8", cache_blocks=0),
               dict(kv_cache="fp8", prefill_chunk=0)):
        with pytest.raises(ValueError):
            FastDecoder(model, CPU, **kw)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 32, 1, 32, CPU, fmt="fp16")
    dec = FastDecoder(model, CPU)
    with pytest.raises(ValueError):
        dec.run_step(torch.tensor([1]), torch.tensor([0]), torch.tensor([1]))


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
def test_unsupported_head_dim_is_refused():
    with pytest.raises(Unsupported, match="head_dim"):
        FastDecoder(_model(hidden_size=64, attention_heads=4), torch.device("cuda"), kv_cache="fp8")


@pytest.mark.gpu
@pytest.mark.skipif(not cuda_ready(), reason="needs a B200")
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("layout", [dict(), dict(hidden_size=128), dict(hidden_size=512, kv_heads=2),
                                    dict(norm_type="layernorm", position_embedding="learned", attention_bias=True)])
def test_native_paged_decoder_matches_the_cpu_oracle(layout, fmt):
    from quantaweave_b200.ops import ext

    # every token goes to both experts: with fewer, bf16 against fp32 changes a token's experts now and then (with the dense
    # cache too), which moves its logits by a tenth of their range
    model = _model(num_experts=2, top_k=2, **layout)
    prompts = torch.randint(0, 512, (4, 60), generator=torch.Generator().manual_seed(3))
    cpu = FastDecoder(model, CPU, max_batch=4, kv_cache=fmt, cache_block=16)
    cpu._prefill(prompts[:, :50])
    want = [cpu.run_step(prompts[:, i], torch.full((4,), i)).clone() for i in range(50, 60)]
    model = model.cuda()
    dec = FastDecoder(model, torch.device("cuda"), max_batch=4, kv_cache=fmt, cache_block=16, prefill_chunk=32)
    assert dec.uses_graph
    dec._prefill(prompts[:, :50].cuda())
    for i in range(50, 60):
        got = dec.run_step(prompts[:, i].cuda(), torch.full((4,), i, device="cuda"))
        assert _close(got, want[i - 50]), i
    assert dec.generate(prompts.cuda(), 8).shape == (4, 8)
    # requests of their own lengths in one step, one left out
    dec.cache.clear()
    for row, n in ((0, 20), (2, 33), (3, 1)):
        dec._prefill(prompts[row:row + 1, :n].cuda(), first_row=row)
    tokens = torch.stack([prompts[0, 20], prompts[2, 33], prompts[3, 1], torch.tensor(0)]).cuda()
    got = dec.run_step(tokens, torch.tensor([20, 0, 33, 1], device="cuda"), torch.tensor([1, 0, 1, 1], device="cuda")).clone()
    for i, (row, n) in enumerate(((0, 20), (2, 33), (3, 1))):
        one = FastDecoder(model, torch.device("cuda"), kv_cache=fmt, cache_block=16)
        assert _close(got[i], one.feed(prompts[row, : n + 1].tolist()))
    assert ext().read_status(True) == 0
