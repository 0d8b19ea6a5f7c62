"""Sampling of batches whose rows take a work-group each however long they are, of the longest chunks, and past 32 bits:
the same tokens and probabilities as the rows of smaller batches, bit for bit, and some rows against 64 bits."""

import pytest
import torch

from ananta_ocr_amd import sampling
from test_gpu_sample import DEV, SETTINGS, _check, _logits

pytestmark = pytest.mark.gpu


def _settings(R):
    t, k, p, m = (list(y) for y in zip(*(SETTINGS[i % len(SETTINGS)] for i in range(R))))
    return (torch.tensor(t, device=DEV), torch.tensor(k, dtype=torch.int32, device=DEV), torch.tensor(p, device=DEV),
            torch.tensor(m, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, V", [(256, 32769), (300, 50001), (700, 40000)])
def test_long_rows_of_large_batches(R, V, dtype):
    x, u = _logits(R, V, R)
    x, u, how = x.to(dtype).to(DEV), torch.tensor(u).to(DEV), _settings(R)
    x[5] = 1.0                                        # more tokens of one logit than are listed
    x[6, :V // 2] = -float("inf")
    token, probs = sampling.sample(x, u, *how, return_probs=True)
    assert torch.equal(sampling.sample(x, u, *how), token)
    for r0 in range(0, R, 100):
        some = slice(r0, min(r0 + 100, R))
        t, p = sampling.sample(x[some], u[some], *(y[some] for y in how), return_probs=True)
        assert torch.equal(t, token[some]) and torch.equal(p, probs[some])
    _check(x[:14].cpu(), u[:14].tolist(), *(y[:14].tolist() for y in how))


@pytest.mark.parametrize("R", [64, 65, 127, 255])
def test_chunks_of_the_largest_vocabulary(R):
    """From sixteen chunks a row down to four, of up to 2^18 tokens."""
    V = 2 ** 20 - 3
    g = torch.Generator(device=DEV).manual_seed(R)
    x = (2.5 * torch.randn(R, V, generator=g, device=DEV)).bfloat16()
    x[:, V - 1] = 9.5
    u, how = torch.rand(R, generator=g, device=DEV), _settings(R)
    u[:5] = 1.0                                       # the last token that stays
    token, probs = sampling.sample(x, u, *how, return_probs=True)
    for r in (0, 1, 4, R // 2, R - 1):
        some = slice(r, r + 1)
        t, p = sampling.sample(x[some], u[some], *(y[some] for y in how), return_probs=True)
        assert torch.equal(t, token[some]) and torch.equal(p, probs[some])
    for r in (2, R - 2):
        _check(x[r:r + 1].cpu(), u[r:r + 1].tolist(), *(float(y[r]) if y.is_floating_point() else int(y[r]) for y in how))


def test_rows_past_32_bits():
    """More than 2^31 logits."""
    R, V = 2 ** 11 + 3, 2 ** 20
    x = torch.empty(R, V, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    x[:4] = (2.5 * torch.randn(4, V, generator=g, device=DEV)).bfloat16()
    x[4:] = x[0]
    x[-3:] = (2.5 * torch.randn(3, V, generator=g, device=DEV)).bfloat16()
    u, how = torch.rand(R, generator=g, device=DEV), _settings(R)
    token = sampling.sample(x, u, *how)
    for some in (slice(0, 4), slice(R - 3, R)):
        assert torch.equal(sampling.sample(x[some].clone(), u[some], *(y[some] for y in how)), token[some])
