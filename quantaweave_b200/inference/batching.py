"""Continuous batching: concurrent generation requests share the decode steps of one ``FastDecoder``.

The reference server runs one request at a time behind an ``asyncio.Lock`` (``src/serve_quantweave.py:211-354``)
and its decoder is batch-1 (``src/fast_decode.py:86-379``). Here the decoder's ``max_batch`` cache rows are slots:

* ``submit`` queues a request (prompt ids, token budget, sampling settings, seed, stop ids, optional per-token
  callback);
* ``step`` admits queued requests into free slots — each prompt is prefilled into its own cache row — then runs ONE
  decode step over all slots (the full batch, so the captured CUDA graph replays), samples every active row with its
  own settings and generator, delivers the token and retires rows that hit a stop id or their budget. Idle slots
  decode a dummy token at position 0 of their own row, which the next request's prefill overwrites.

Requests therefore join and leave between steps without waiting for each other, and a step costs the same whether
one or ``max_batch`` requests are active.

With a block-wise cache (``FastDecoder(kv_cache="fp8")``) the slots share a pool of blocks: a request is admitted when the
blocks of its prompt and budget fit beside those promised to the others, idle slots hold none, and a retired request's
return to the pool. Penalties and grammar masks (``GenerationRequest``) are applied to the step's logits on the device in one
pass (``ops.logits``).
"""

from __future__ import annotations

import threading
from collections import deque
from dataclasses import dataclass, field
from typing import Callable, Optional

import torch

from .fast_decode import FastDecoder, filter_logits


PENALTY_LIMIT = 1e6


@dataclass
class GenerationRequest:
    prompt: list
    max_new: int
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    seed: int = 0
    stop_ids: tuple = ()
    on_token: Optional[Callable[[int], None]] = None
    logit_bias: Optional[torch.Tensor] = None  # added to the logits before sampling (e.g. -inf on invalid ids)
    repetition_penalty: float = 1.0  # positive logits of ids seen (prompt and generated) divided by it, others multiplied
    frequency_penalty: float = 0.0   # subtracted per occurrence among the generated ids
    presence_penalty: float = 0.0    # subtracted once for each generated id
    allowed: Optional[Callable[[list], torch.Tensor]] = None  # generated ids -> bool [vocab]: what a grammar lets follow
    cancelled: bool = False  # set (e.g. by ``on_token`` on a text stop string) to retire the request after this token
    # results
    tokens: list = field(default_factory=list)
    finish_reason: Optional[str] = None
    done: threading.Event = field(default_factory=threading.Event)

    @property
    def penalised(self) -> bool:
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    def wait(self, timeout: Optional[float] = None) -> list:
        if not self.done.wait(timeout):
            raise TimeoutError("generation did not finish in time")
        return self.tokens


class ContinuousBatcher:
    def __init__(self, decoder: FastDecoder) -> None:
        if decoder.native and not hasattr(decoder, "_C"):
            from ..ops import ext

            decoder._C = ext()  # the native prefill's RoPE / attention entry points
        self.decoder = decoder
        self.slots = decoder.max_batch
        self.active: dict[int, GenerationRequest] = {}
        self.waiting: deque = deque()
        self.lock = threading.Lock()
        self._position = [0] * self.slots
        self._next_token = [0] * self.slots
        self._generators: dict[int, torch.Generator] = {}
        # block-wise cache: blocks promised to each slot's request, and slots that may still hold blocks of no active request
        self._blocks = [0] * self.slots
        self._unreleased: set = set()
        self.steps = 0

    # ---- queue --------------------------------------------------------------------------------------------
    def submit(self, request: GenerationRequest) -> GenerationRequest:
        if not request.prompt:
            raise ValueError("a request needs at least one prompt token")
        if request.max_new < 1:
            raise ValueError("max_new must be positive")
        if len(request.prompt) + request.max_new > self.decoder.capacity:
            raise ValueError(f"prompt ({len(request.prompt)}) + max_new ({request.max_new}) exceed the decoder "
                             f"context {self.decoder.capacity}")
        # NaN fails these too; within them no logit leaves the range of 32-bit numbers
        if not 0 < request.repetition_penalty:
            raise ValueError("repetition_penalty must be positive")
        if not 1 / PENALTY_LIMIT <= request.repetition_penalty <= PENALTY_LIMIT:
            raise ValueError(f"repetition_penalty must lie between {1 / PENALTY_LIMIT:g} and {PENALTY_LIMIT:g}")
        for name in ("frequency_penalty", "presence_penalty"):
            if not abs(getattr(request, name)) <= PENALTY_LIMIT:
                raise ValueError(f"{name} must be a number of at most {PENALTY_LIMIT:g} in magnitude")
        cache = self.decoder.cache
        if cache is not None and self._blocks_of(request) > cache.blocks:
            raise ValueError(f"prompt ({len(request.prompt)}) + max_new ({request.max_new}) need {self._blocks_of(request)} "
                             f"cache blocks, the pool has {cache.blocks}")
        with self.lock:
            self.waiting.append(request)
        return request

    def _blocks_of(self, request: GenerationRequest) -> int:
        return self.decoder.cache.blocks_for(len(request.prompt) + request.max_new)

    def withdraw(self, request: GenerationRequest) -> bool:
        """Take a request that has not reached a slot yet back out of the queue; False once it is decoding."""
        with self.lock:
            try:
                self.waiting.remove(request)
            except ValueError:
                return False
        request.finish_reason = "withdrawn"
        request.done.set()
        return True

    def pending(self) -> int:
        with self.lock:
            return len(self.waiting) + len(self.active)

    # ---- scheduling ---------------------------------------------------------------------------------------
    def _admit(self) -> None:
        if not self.active and self.waiting:  # the decoder may have been used for something else meanwhile
            self._unreleased.update(range(self.slots))
        if self._unreleased:
            if self.decoder.cache is not None:
                self.decoder.cache.release_rows(sorted(self._unreleased - set(self.active)))
            self._unreleased.clear()
        while True:
            with self.lock:
                free = [s for s in range(self.slots) if s not in self.active]
                if not free or not self.waiting:
                    return
                if self.decoder.cache is not None:
                    promised = sum(self._blocks[s] for s in self.active)
                    if promised + self._blocks_of(self.waiting[0]) > self.decoder.cache.blocks:
                        return  # the next in line waits for blocks, and the others behind it
                request = self.waiting.popleft()
            slot = free[0]
            if self.decoder.cache is not None:
                self._blocks[slot] = self._blocks_of(request)
            prompt = list(request.prompt)
            try:
                self.decoder._prefill(torch.tensor([prompt[:-1]], dtype=torch.long), first_row=slot)
            except BaseException as exc:
                # the request left the queue but never reached a slot: finish it here so its waiter returns
                self._unreleased.add(slot)
                request.finish_reason = f"error: {exc}"
                request.done.set()
                raise
            self._position[slot] = len(prompt) - 1
            self._next_token[slot] = prompt[-1]
            self._generators[slot] = torch.Generator().manual_seed(request.seed)
            with self.lock:
                self.active[slot] = request

    def _masks(self, rows: list, failed: dict) -> dict:
        """``{slot: bool [vocab]}`` of the active rows with a grammar; an error goes to ``failed[slot]``."""
        masks = {}
        for slot in rows:
            request = self.active[slot]
            if request.allowed is None:
                continue
            try:
                mask = torch.as_tensor(request.allowed(request.tokens)).cpu().bool()
                if mask.shape != (self.decoder.vocab,):
                    raise ValueError(f"the grammar's mask must be [{self.decoder.vocab}], got {list(mask.shape)}")
                masks[slot] = mask
            except Exception as exc:  # noqa: BLE001 - a request's own callback: it alone ends
                failed[slot] = exc
        return masks

    def _processed(self, logits: torch.Tensor, rows: list, failed: dict) -> torch.Tensor:
        """Penalties and grammar masks of the active rows' requests, in one pass on the logits' device."""
        requests = [self.active[s] for s in rows]
        if not any(r.penalised or r.allowed is not None for r in requests):
            return logits
        from ..ops.logits import pack_mask, process_logits

        dev, kw = logits.device, {}
        if any(r.penalised for r in requests):
            seen = [list(r.prompt) + r.tokens for r in requests]
            length = max(len(ids) for ids in seen)
            history = torch.tensor([ids + [0] * (length - len(ids)) for ids in seen], dtype=torch.int32)
            lens = torch.tensor([[len(ids) for ids in seen], [len(r.prompt) for r in requests]], dtype=torch.int32).to(dev)
            penalties = torch.tensor([[r.repetition_penalty for r in requests], [r.frequency_penalty for r in requests],
                                      [r.presence_penalty for r in requests]]).to(dev)
            kw.update(history=history.to(dev), history_lens=lens[0], prompt_lens=lens[1], repetition=penalties[0],
                      frequency=penalties[1], presence=penalties[2])
        masks = self._masks(rows, failed)
        if masks:
            which = {slot: i for i, slot in enumerate(masks)}
            kw.update(mask=pack_mask(torch.stack(list(masks.values()))).to(dev),
                      mask_rows=torch.tensor([which.get(s, -1) for s in rows], dtype=torch.int32).to(dev))
        return process_logits(logits, **kw)

    def _sample(self, logits: torch.Tensor, request: GenerationRequest, generator: torch.Generator) -> int:
        if request.logit_bias is not None:
            logits = logits + request.logit_bias
        if request.temperature <= 0:
            token = int(logits.argmax())
            if (request.allowed is not None or request.logit_bias is not None) and logits[token].item() == float("-inf"):
                raise ValueError("no token is allowed")
            return token
        filtered = filter_logits(logits[None] / request.temperature, request.top_k, request.top_p)[0]
        return int(torch.multinomial(filtered.softmax(-1), 1, generator=generator))

    @torch.no_grad()
    def step(self) -> int:
        """Admit queued requests, advance every active one by one token; returns the number still active."""
        self._admit()
        with self.lock:
            rows = sorted(self.active)
        if not rows:
            return 0
        dev = self.decoder.device
        positions = torch.tensor([self._position[s] if s in rows else 0 for s in range(self.slots)],
                                 dtype=torch.int32, device=dev)
        if self.decoder.cache is not None:  # the active rows only, in slot order; idle slots have no token
            tokens = [self._next_token[s] for s in rows] + [0] * (self.slots - len(rows))
            new = torch.tensor([int(s in rows) for s in range(self.slots)], dtype=torch.int32, device=dev)
            # the blocks promised to the active requests suffice
            logits = self.decoder._run_step(torch.tensor(tokens, device=dev), positions, new)[: len(rows)]
        else:
            tokens = torch.tensor([self._next_token[s] if s in rows else 0 for s in range(self.slots)], device=dev)
            logits = self.decoder.run_step(tokens, positions)[rows]
        failed: dict = {}  # a request whose grammar or sampling fails ends alone
        logits = self._processed(logits.float(), rows, failed).cpu()
        self.steps += 1
        for i, slot in enumerate(rows):
            request = self.active[slot]
            if slot not in failed:
                try:
                    token = self._sample(logits[i], request, self._generators[slot])
                except Exception as exc:  # noqa: BLE001
                    failed[slot] = exc
            if slot in failed:
                self._retire(slot, f"error: {failed[slot]}")
                continue
            request.tokens.append(token)
            if request.on_token is not None:
                request.on_token(token)
            self._position[slot] += 1
            self._next_token[slot] = token
            reason = None
            if request.cancelled or token in request.stop_ids:
                reason = "stop"
            elif len(request.tokens) >= request.max_new or self._position[slot] + 1 >= self.decoder.capacity:
                reason = "length"
            if reason is not None:
                self._retire(slot, reason)
        with self.lock:
            return len(self.active)

    def _retire(self, slot: int, reason: str) -> None:
        request = self.active[slot]
        request.finish_reason = reason
        with self.lock:
            del self.active[slot]
        if self.decoder.cache is not None:
            self.decoder.cache.release_rows([slot])
        request.done.set()

    def run_until_idle(self) -> None:
        while self.pending():
            self.step()


class BatchingWorker:
    """A background thread that keeps stepping a ``ContinuousBatcher`` while requests are queued or active."""

    def __init__(self, batcher: ContinuousBatcher) -> None:
        self.batcher = batcher
        self._wake = threading.Event()
        self._stop = threading.Event()
        self.error: Optional[BaseException] = None
        self._thread = threading.Thread(target=self._loop, name="qw-batcher", daemon=True)
        self._thread.start()

    def submit(self, request: GenerationRequest) -> GenerationRequest:
        if self._stop.is_set():
            raise RuntimeError("the batching worker is closed")
        self.batcher.submit(request)
        self._wake.set()
        return request

    def _loop(self) -> None:
        while not self._stop.is_set():
            if not self.batcher.pending():
                self._wake.wait(0.05)
                self._wake.clear()
                continue
            try:
                self.batcher.step()
            except BaseException as exc:  # noqa: BLE001 - fail every waiting request instead of hanging them
                self.error = exc
                self._fail_all(f"error: {exc}")

    def _fail_all(self, reason: str) -> None:
        with self.batcher.lock:
            stuck = list(self.batcher.active.values()) + list(self.batcher.waiting)
            self.batcher._unreleased.update(self.batcher.active)
            self.batcher.active.clear()
            self.batcher.waiting.clear()
        for request in stuck:
            request.finish_reason = reason
            request.done.set()

    def close(self) -> None:
        """Stop stepping; requests still queued or in flight finish with reason ``closed``."""
        self._stop.set()
        self._wake.set()
        self._thread.join(timeout=5)
        self._fail_all("closed")
