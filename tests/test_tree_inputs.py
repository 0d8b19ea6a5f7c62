"""Tree steps and page calls on the host: batches without requests, tables written in place.  No GPU
calls."""

import pytest
import torch

from ananta_ocr_amd import kv_pages, pipeline

I32 = torch.int32


@pytest.mark.parametrize("width", [128, 64])
@pytest.mark.parametrize("rows", [0, 5])
def test_steps_without_requests(width, rows):
    """No request at all, with and without the rows of a batch of fixed size."""
    state = pipeline.KBarPageCache(4, width, "cpu")
    out, (idx, bias, valid), pos = pipeline.tree_step(
        state, torch.zeros(rows, 2, 128), torch.zeros(4, 64, 2, 128), torch.zeros(4, 64, 2, 128),
        torch.zeros(rows, width), 64, 1, 1.0, 1e-4, 1.0, 3, 4, torch.zeros(0, 6, dtype=I32),
        torch.zeros(0, dtype=I32), torch.zeros(1, dtype=I32), torch.zeros(rows, dtype=I32), 4,
        return_routing=True)
    assert out.shape == (rows, 2, 128) and out.dtype == torch.bfloat16
    assert idx.shape == bias.shape == valid.shape == (rows, 3) and pos.shape == (rows,)
    assert not valid.any()
