"""The batching server over the block-wise 8-bit KV cache, and its request penalties (CPU forms)."""

import asyncio

import pytest
import torch
from fastapi import HTTPException
from test_tools_cpu import _train

from quantaweave_b200.tools.serve import GenerateRequest, Server


@pytest.fixture(scope="module")
def checkpoint(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("serve")
    _train(tmp, steps=1, hidden_size=64)
    return tmp / "out"


def _generate(server, **options):
    return asyncio.run(server.generate(GenerateRequest(prompt="the", tokens=12, temperature=0.0, stop=[], **options)))


@pytest.mark.parametrize("kv_cache", ["fp8", "int8"])
def test_a_server_with_the_block_wise_cache_answers_and_describes_it(checkpoint, kv_cache):
    server = Server(checkpoint, None, torch.device("cpu"), "fp32", batching=2, kv_cache=kv_cache, cache_blocks=8)
    try:
        assert kv_cache in server.info()["batching_cache"]
        first, second = _generate(server), _generate(server)
        assert first["tokens"] == 12 and first["text"] == second["text"]  # the blocks of the first were given again
    finally:
        server.close()


def test_penalties_change_what_a_batched_request_gets_and_nothing_else(checkpoint):
    server = Server(checkpoint, None, torch.device("cpu"), "fp32", batching=2, kv_cache="fp8")
    try:
        plain = _generate(server)
        free = _generate(server, presence_penalty=100.0)  # no id twice while others are left
        assert len(set(free["text"])) == len(free["text"]) > 1
        assert _generate(server)["text"] == plain["text"]
    finally:
        server.close()


def test_penalties_without_batching_are_refused(checkpoint):
    server = Server(checkpoint, None, torch.device("cpu"), "fp32")
    try:
        assert server.info()["batching_cache"] is None
        with pytest.raises(HTTPException) as refused:
            _generate(server, repetition_penalty=1.2)
        assert refused.value.status_code == 422
    finally:
        server.close()
