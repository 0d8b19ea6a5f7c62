"""Attention of trees (tree.attn_tree) where single bits count: bf16 outputs."""

import pytest
import torch

from test_gpu_tree import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("case", [
    ([300], [8], 2, 2, 64, 2, 4), ([333, 1000], [13, 32], 10, 2, 32, 4, 12),
    ([640, 64], [33, 64], 4, 1, 64, 1, 3), ([5000, 3000], [32, 20], 4, 4, 64, 4, 16),
    ([5000, 2100], [64, 40], 4, 4, 64, 4, 16)])
def test_bf16_outputs_are_the_fp32_ones_rounded_once(case):
    """Nothing before the output goes by its type: in every height of the row tiles and with one
    split and several, the bf16 output is the fp32 one to the nearest bf16."""
    c = _case(*case, seed=3)
    full, lse = _run(c, return_lse=True)
    half, lse16 = _run(c, return_lse=True, out_dtype=torch.bfloat16)
    assert torch.equal(half, full.bfloat16()) and torch.equal(lse, lse16)
