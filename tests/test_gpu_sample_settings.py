"""Types and extremes of the sampling's settings (sampling.sample, sampling.token_probs)."""

import pytest
import torch

from ananta_ocr_amd import sampling
from test_gpu_sample import DEV, _logits

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
