"""What kv_pages.step_rows refuses.  No GPU calls."""

import pytest
import torch

from ananta_ocr_amd import kv_pages

I32 = torch.int32


def test_refusals():
    table, two = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    for args, err in (((table[0], two, two, 8, 4, 4), ValueError), ((table, two[:1], two, 8, 4, 4), ValueError),
                      ((table, two, two[:1], 8, 4, 4), ValueError), ((table, two, two, 0, 4, 4), ValueError),
                      ((table, two, two, 8, -1, 4), ValueError), ((table, two, two, 8, 4, -1), ValueError),
                      ((table, two, two, 8, 4, 2 ** 31), ValueError),
                      ((table, two, two, 8, 4, 4, two[:1]), ValueError),
                      ((table, two, two, 8, 4, 4), ValueError)):        # (last: tensors of the CPU)
        with pytest.raises(err):
            kv_pages.step_rows(*args)
    many = torch.zeros(8193, dtype=I32)
    with pytest.raises(NotImplementedError):
        kv_pages.step_rows(many[:, None], many, many, 8, 4, 4)
