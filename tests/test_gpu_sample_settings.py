"""Types and extremes of the sampling's settings (sampling.sample, sampling.token_probs)."""

import math

import pytest
import torch

from ananta_ocr_amd import sampling
from test_gpu_sample import DEV, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32,
                                   torch.int64])
def test_top_k_of_any_whole_numbers(dtype):
    x, u = _logits(4, 900, 41)
    k = [0, 1, 50, 120]
    x, u = x.to(DEV), torch.tensor(u).to(DEV)
    token, probs = sampling.sample(x, u, 0.9, torch.tensor(k).to(dtype).to(DEV), 0.9, return_probs=True)
    for r in range(4):
        t, p = sampling.sample(x[r:r + 1], u[r:r + 1], 0.9, k[r], 0.9, return_probs=True)
        assert torch.equal(t, token[r:r + 1]) and torch.equal(p, probs[r:r + 1])
    if dtype.is_signed:
        assert torch.equal(sampling.sample(x, u, 0.9, torch.full((4,), -3, dtype=dtype, device=DEV)),
                           sampling.sample(x, u, 0.9, 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 300, 5000, 40000])
@pytest.mark.parametrize("t", [math.inf, 3e38, 1e38, 2e37, 1e36])
def test_logits_further_apart_than_the_largest_number(V, dtype, t):
    """Temperatures at which the type's lowest value still has a weight beside its highest."""
    g = torch.Generator().manual_seed(V)
    top = torch.finfo(dtype).max
    x = (2 * torch.rand(4, V, generator=g, dtype=torch.float64) - 1) * top
    x[0, ::3], x[0, 1::3], x[0, 2::3] = top, -top, 0.0
    x[1, V // 2], x[1, V // 3] = top, -top
    x[2, 1:] = -top
    x = x.to(dtype)
    u = torch.rand(4, generator=g).tolist()
    for k, p, m in ((0, 1.0, 0.0), (V // 2, 1.0, 0.0), (0, 0.6, 0.0), (V // 2 + 1, 0.7, 0.0), (0, 1.0, 0.3),
                    (0, 0.9, 1e-4), (0, 1.0, 1.0)):
        _check(x, u, t, k, p, m)
