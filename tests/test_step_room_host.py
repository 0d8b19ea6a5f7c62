"""What kv_pages.PagePool.reserve_step and its entry point refuse.  No GPU calls."""

import pytest
import torch

from ananta_ocr_amd import kv_pages
from test_capi import ERR_INVALID, _call

I32 = torch.int32


class _Caches:
    """What a pool asks of its caches."""
    device, num_pages, page_size = torch.device("cpu"), 4, 8


def test_refusals():
    pool, two = kv_pages.PagePool(_Caches, 2, 3), torch.zeros(2, dtype=I32)
    for args, err in (((two[:1], 4), ValueError), ((two, -1), ValueError), ((two, 2 ** 31), ValueError),
                      ((two, 4), ValueError)):                   # (last: tensors of the CPU)
        with pytest.raises(err):
            pool.reserve_step(*args)
    pool.table = torch.zeros(1, 1, dtype=I32).expand(2, 2 ** 28)
    with pytest.raises(NotImplementedError):
        pool.reserve_step(two, 4)


def test_entry_point():
    for kw in (dict(R=-1, rows=4), dict(R=2, rows=-1), dict(R=2, rows=4, lens=None),
               dict(R=2, rows=4, new_lens=None)):
        assert _call("dash_step_lens", **{**dict(stream=None), **kw}) == ERR_INVALID
    assert _call("dash_step_lens", R=0, rows=4, stream=None) == 0
