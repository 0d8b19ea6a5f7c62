"""Types that the attention of shared prompts refuses.  No GPU calls."""

import contextlib

import pytest
import torch

from ananta_ocr_amd import pipeline, shared_prefix

I32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("other", [torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("which", ["q", "k", "v", "qkv"])
def test_no_casts(monkeypatch, which, other):
    """A cast would round the queries, or copy the whole pool at every call."""
    monkeypatch.setattr(shared_prefix, "_device", lambda *a: contextlib.nullcontext())
    x = dict(q=torch.zeros(3, 4, 128), k=torch.zeros(5, 16, 2, 128), v=torch.zeros(5, 16, 2, 128))
    x = {n: t.to(other if n in which else torch.bfloat16) for n, t in x.items()}
    with pytest.raises(NotImplementedError, match="bf16"):
        shared_prefix.attn_shared(x["q"], x["k"], x["v"], torch.zeros(2, 3, **I32), torch.zeros(2, **I32),
                                  torch.tensor([0, 1, 3], **I32), None, None, 0.1)


def test_a_layer_refuses_before_it_writes():
    x = torch.zeros(3, 4, 128, dtype=torch.float16)
    caches = [torch.zeros(5, 16, 4, 128, dtype=torch.float16) for _ in range(2)]
    step = pipeline.StepRows(*[torch.zeros(3, **I32)] * 6)
    with pytest.raises(NotImplementedError, match="bf16"):
        pipeline.shared_step(step, x, x, x, *caches, torch.zeros(3, 2, **I32), torch.zeros(64))
