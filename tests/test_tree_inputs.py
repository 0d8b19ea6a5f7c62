"""Tree steps and page calls on the host: batches without requests, tables written in place.  No GPU
calls."""

import pytest
import torch

from ananta_ocr_amd import kv_pages, pipeline, tree

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


def test_page_calls_refuse_rows_that_overlap():
    """One row for all, or rows that share entries, cannot be written in place; a column of a wider
    table, or a table of one row of any stride, can."""
    refs, lens = torch.zeros(9, dtype=I32), torch.zeros(3, dtype=I32)
    for table in (torch.zeros(1, 4, dtype=I32).expand(3, 4),
                  torch.zeros(20, dtype=I32).as_strided((3, 4), (3, 1))):
        for f, more in ((kv_pages.fork_pages, (lens[:1], lens[:1])), (kv_pages.reserve_pages, (lens,)),
                        (kv_pages.free_pages, (lens,))):
            with pytest.raises(ValueError, match="overlap"):
                f(refs, table, lens, *more, 8)
    for table in (torch.zeros(3, 7, dtype=I32)[:, 2:6], torch.zeros(3, 5, dtype=I32)[:, 1:2],
                  torch.zeros(3, 4, dtype=I32)):
        with pytest.raises(ValueError, match="GPU"):
            kv_pages.reserve_pages(refs, table, lens, lens, 8)
    with pytest.raises(ValueError, match="GPU"):
        kv_pages.reserve_pages(refs, torch.zeros(1, 4, dtype=I32).expand(1, 4), lens[:1], lens[:1], 8)


def test_attention_refuses_tables_of_more_tokens_than_32_bits():
    """A row of the table for 2^32 tokens and a few more would be taken for the few."""
    a = dict(q=torch.zeros(5, 4, 128), k=torch.zeros(3, 64, 2, 128), v=torch.zeros(3, 64, 2, 128), idx=None,
             bias=None, valid=None, mask=torch.zeros(5, 1, dtype=torch.int64), depth=torch.zeros(5, dtype=I32),
             context_lens=torch.zeros(2, dtype=I32), cu_seqlens_q=torch.tensor([0, 1, 5]), max_query_len=4,
             block_size=64, local_window=128, scale=0.1, page_size=64)
    for pages in (2 ** 26 + 16, 2 ** 25):
        with pytest.raises(NotImplementedError):
            tree.attn_tree(**a, block_table=torch.zeros(1, 1, dtype=I32).expand(2, pages))
    with pytest.raises(ValueError, match="GPU"):
        tree.attn_tree(**a, block_table=torch.zeros(1, 1, dtype=I32).expand(2, 2 ** 25 - 1))
