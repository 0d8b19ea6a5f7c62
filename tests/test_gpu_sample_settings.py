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


@pytest.mark.parametrize("V", [700, 32000, 131072])
@pytest.mark.parametrize("spread, t", [(2.5, 1.0), (2.5, 0.05), (40.0, 1.0), (0.01, 1.0)])
def test_what_whole_number_weights_leave_out(V, spread, t):
    """Against a softmax that leaves no token out.  With s = 62 - ceil(log2 V), 51 at most, a weight below
    2^-(s + 1) of the best token's is none: that much of a probability at most.  The V roundings of 2^-(s + 1) in
    the sum, which is 1 at least, are V 2^-(s + 1) of the others, beside half a step of 32 bits and the
    reference's own 2^-40."""
    x, _ = _logits(3, V, V + 1, spread=spread)
    z = x.double() / torch.tensor(t, dtype=torch.float32).double()
    w = (z - z.max(1, keepdim=True).values).exp()
    want = w / w.sum(1, keepdim=True)
    s = min(51, 62 - (V - 1).bit_length())
    got = sampling.token_probs(x.to(DEV), t).double().cpu()
    tol = want * (2.0 ** -24 + V * 2.0 ** -(s + 1) + 2.0 ** -40) + 2.0 ** -(s + 1)
    assert bool(((got - want).abs() <= tol).all())
    # the k tokens of most weight
    order = want.sort(1, descending=True)
    k = min(V // 2, 40)
    kept = torch.zeros_like(want).scatter(1, order.indices[:, :k], order.values[:, :k])
    kept /= kept.sum(1, keepdim=True)
    got = sampling.token_probs(x.to(DEV), t, k).double().cpu()
    assert bool(((got - kept).abs() <= kept * (2.0 ** -24 + 2.0 ** -s * V + 2.0 ** -39) + 2.0 ** -s).all())
