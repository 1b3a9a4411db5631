"""The block-wise 8-bit KV cache at its edges: held scales that are none, numbers far below their row's largest, no heads,
offsets that do not fit, inputs that ask for gradients."""

import math

import pytest
import torch

from conftest import cuda_ready
from quantaweave_b200.ops import kv_cache as kvc

GPU = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ready(), reason="needs a B200")]
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("held", [0.0, math.nan, math.inf])
def test_a_held_scale_that_is_none_sets_no_scale(held, fmt, device):
    """A cache that was never written holds zeros, its scales as well: a write into the middle of a block takes the new
    numbers' own scale."""
    x = torch.tensor([0.75, -0.5]).repeat(16)[None, None].bfloat16()
    kc, vc = (torch.zeros(1, 1, 16, 32, dtype=kvc.FORMATS[fmt], device=device) for _ in range(2))
    ks, vs = (torch.full((1, 1), held, device=device) for _ in range(2))
    kvc.append_kv(x.to(device), x.to(device), torch.tensor([5], dtype=torch.int32, device=device), kc, vc, ks, vs)
    scale = 2.0 ** (-9 if fmt == "fp8" else -7)  # 0.75 = 384 * 2^-9 = 96 * 2^-7
    for codes, scales in ((kc, ks), (vc, vs)):
        assert scales.tolist() == [[scale]]
        assert torch.equal(codes[0, 0, 5].cpu().double() * scale, x[0, 0].double())
