"""What the sampling and shared-prompt calls refuse.  No GPU calls."""

import pytest
import torch

from ananta_ocr_amd import sampling, shared_prefix

I32 = torch.int32


def test_sampling_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for args, kw, err in (((x[0], u), {}, ValueError), ((x[:, :0], u), {}, ValueError), ((x, u[:1]), {}, ValueError),
                          ((x, None), {}, ValueError), ((x, u, u[:1]), {}, ValueError),
                          ((x, u, 1.0, torch.zeros(3, dtype=I32)), {}, ValueError),
                          ((x, u, 1.0, torch.zeros(2)), {}, ValueError), ((x, u, 1.0, 0, u[:1]), {}, ValueError),
                          ((x, u, 1.0, 0, 1.0, u[:1]), {}, ValueError),
                          ((x, u), dict(return_probs=True, probs_dtype=torch.float64), NotImplementedError),
                          ((torch.zeros(1, 1).expand(1, 2 ** 20 + 1), u[:1]), {}, NotImplementedError),
                          ((x, u), {}, ValueError)):             # (last: tensors of the CPU)
        with pytest.raises(err):
            sampling.sample(*args, **kw)
    with pytest.raises(NotImplementedError):
        sampling.token_probs(x, dtype=torch.int32)


def test_shared_prompt_refusals():
    q, k = torch.zeros(3, 4, 128), torch.zeros(5, 16, 2, 128)
    table, two = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    cu = torch.tensor([0, 1, 3], dtype=I32)
    gr, pre = torch.tensor([0, 2], dtype=I32), torch.zeros(1, dtype=I32)
    ok = dict(q=q, k=k, v=k, block_table=table, context_lens=two, cu_seqlens_q=cu, cu_groups=gr, prefix_lens=pre,
              scale=0.1)
    for bad, err in ((dict(q=q[0]), ValueError), (dict(v=k[:4]), ValueError), (dict(q=torch.zeros(3, 3, 128)), ValueError),
                     (dict(q=torch.zeros(3, 4, 64)), ValueError), (dict(block_table=table[0]), ValueError),
                     (dict(context_lens=two[:1]), ValueError), (dict(cu_seqlens_q=two), ValueError),
                     (dict(cu_groups=None), ValueError), (dict(prefix_lens=None), ValueError),
                     (dict(prefix_lens=two), ValueError), (dict(cu_groups=gr[None]), ValueError),
                     (dict(out_dtype=torch.float16), NotImplementedError),
                     (dict(k=k[:, :0], v=k[:, :0]), ValueError),
                     (dict(block_table=torch.zeros(1, 1, dtype=I32).expand(2, 2 ** 27)), NotImplementedError),
                     (dict(block_table=torch.zeros(8193, 1, dtype=I32), context_lens=torch.zeros(8193, dtype=I32),
                           cu_seqlens_q=torch.zeros(8194, dtype=I32)), NotImplementedError),
                     (dict(), ValueError)):                      # (last: tensors of the CPU)
        with pytest.raises(err):
            shared_prefix.attn_shared(**{**ok, **bad})
