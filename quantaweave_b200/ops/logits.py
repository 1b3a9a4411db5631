"""Logits before sampling: penalties for repeated tokens, biases and grammar masks in one pass (``csrc/logits.cu``)."""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import ext, refuse_gradients


def pack_mask(allowed: Tensor) -> Tensor:
    """Bits of ``allowed [..., vocab]`` (bool) as ``process_logits`` reads them: int32 ``[..., ceil(vocab / 32)]``, id
    ``i`` in bit ``i % 32`` of word ``i // 32``."""
    vocab = allowed.size(-1)
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -vocab % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def process_logits(logits: Tensor, *, history: Optional[Tensor] = None, history_lens: Optional[Tensor] = None,
                   prompt_lens: Optional[Tensor] = None, repetition: Optional[Tensor] = None,
                   frequency: Optional[Tensor] = None, presence: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                   bias_rows: Optional[Tensor] = None, mask: Optional[Tensor] = None, mask_rows: Optional[Tensor] = None,
                   out: Optional[Tensor] = None) -> Tensor:
    """``logits [rows, vocab]`` (float32, bfloat16 or float16; any row stride), in this order:

    * ``repetition [rows]`` (> 0): a positive logit is divided by it, another multiplied, for every id among the first
      ``history_lens[r]`` entries of ``history [rows, length]`` (int32);
    * ``frequency [rows]`` times the count, and ``presence [rows]`` once, are subtracted for the ids from entry
      ``prompt_lens[r]`` on (the generated ones; all of them without ``prompt_lens``);
    * ``bias [biases, vocab]`` (float32): row ``bias_rows[r]`` is added, none where that is negative;
    * ``mask [masks, ceil(vocab / 32)]`` (see ``pack_mask``): ids whose bit is 0 in row ``mask_rows[r]`` become -inf.

    Without ``bias_rows`` (``mask_rows``) row ``r`` has bias (mask) row ``r``. Ids outside the vocabulary are ignored. Sums
    are in 32 bits, rounded once. ``out`` may be ``logits`` itself. There is no backward pass: inputs that ask for gradients
    are refused."""
    if logits.is_cuda:
        return ext().process_logits(logits, history, history_lens, prompt_lens, repetition, frequency, presence, bias,
                                    bias_rows, mask, mask_rows, out)
    refuse_gradients("process_logits", logits, repetition, frequency, presence, bias)
    if history is None and not (repetition is None and frequency is None and presence is None):
        raise RuntimeError("process_logits: penalties need the history")
    if history is not None and history_lens is None:
        raise RuntimeError("process_logits: history needs history_lens")
    x = logits.float().clone()
    rows, vocab = x.shape
    for r in range(rows):
        if history is not None:
            ids = history[r, : int(history_lens[r])].long()
            prompt = 0 if prompt_lens is None else int(prompt_lens[r])
            made = ids[max(prompt, 0):]
            ids, made = (i[(i >= 0) & (i < vocab)] for i in (ids, made))
            seen = torch.bincount(ids, minlength=vocab) > 0
            count = torch.bincount(made, minlength=vocab).float()
            if repetition is not None:
                x[r] = torch.where(seen, torch.where(x[r] > 0, x[r] / repetition[r], x[r] * repetition[r]), x[r])
            if frequency is not None:
                x[r] = torch.where(count > 0, x[r] - count * frequency[r], x[r])
            if presence is not None:
                x[r] = torch.where(count > 0, x[r] - presence[r], x[r])
        row = r if bias_rows is None else int(bias_rows[r])
        if bias is not None and 0 <= row < bias.size(0):
            x[r] += bias[row]
        row = r if mask_rows is None else int(mask_rows[r])
        if mask is not None and 0 <= row < mask.size(0):
            bits = (mask[row][:, None] >> torch.arange(32, dtype=torch.int32)) & 1
            x[r] = x[r].masked_fill(bits.flatten()[:vocab] == 0, -math.inf)
    if out is None:
        return x.to(logits.dtype)
    return out.copy_(x)
