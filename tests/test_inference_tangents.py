"""Calls without derivatives refuse inputs that carry a tangent, as they refuse those that require gradients: their
outputs would come without one, which counts as a derivative of 0.  No GPU calls."""

import pytest
import torch
from torch.autograd import forward_ad

from ananta_ocr_amd import rope, sampling, shared_prefix

I32 = dict(dtype=torch.int32)


def test_attention_of_shared_prompts():
    q, k = torch.zeros(3, 4, 128), torch.zeros(5, 16, 2, 128)
    rest = torch.zeros(2, 3, **I32), torch.zeros(2, **I32), torch.tensor([0, 1, 3], **I32), None, None, 0.1
    with forward_ad.dual_level():
        for n in range(3):
            args = [q, k, k]
            args[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(ValueError, match="gradients"):
                shared_prefix.attn_shared(*args, *rest)


def test_rows_of_a_cache():
    x, i, f = torch.zeros(4, 1, 16), torch.arange(4), rope.inv_freq(16)[0]
    caches = torch.zeros(2, 2, 4, 1, 16)
    with forward_ad.dual_level():
        for n in range(3):
            args = [x, x, x]
            args[n] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(ValueError, match="gradients"):
                rope.rope_append(*args, i, i, *caches, f)


def test_probabilities():
    x = torch.zeros(2, 7)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="gradients"):
            sampling.token_probs(x)
        with pytest.raises(ValueError, match="gradients"):
            sampling.sample(x, torch.zeros(2), return_probs=True)
