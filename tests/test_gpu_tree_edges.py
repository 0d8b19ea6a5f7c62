"""Attention of trees (tree.attn_tree) where single bits count: bf16 outputs and biases
that are no numbers."""

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


@pytest.mark.parametrize("case", [
    ([300, 700], [8, 5], 2, 2, 64, 2, 4), ([640], [50], 1, 1, 64, 1, 3), ([640], [100], 2, 1, 32, 1, 3)])
def test_a_bias_that_is_no_number_whatever_its_bits(case):
    """A routed block whose bias is a NaN is a NaN in its row, with the bits of any NaN there is; the
    other rows stay as they are."""
    c = _case(*case, seed=6, bad=False)
    c["idx"][:], c["valid"][:] = -1, True
    nan = torch.tensor([0x7fc00000, -1, 0x7f800001, -0x7fffff], dtype=torch.int32).view(torch.float32)
    T = c["q"].shape[0]
    hit = torch.arange(T) % 3 == 1
    c["idx"][:, 1] = 1
    c["bias"][hit, 1] = nan[torch.arange(T) % 4][hit]
    out, lse = _run(c, return_lse=True)
    want = hit[:, None].expand_as(lse.cpu())
    assert torch.equal(lse.isnan().cpu(), want)
    assert torch.equal(out.isnan().all(-1).cpu(), want) and torch.equal(out.isnan().any(-1).cpu(), want)
