"""Sizes that a launch cannot have (its work-items are counted in 32 bits) are refused before any launch.
No GPU calls."""

import ctypes
import os

import pytest
import torch

from ananta_ocr_amd import _lib
from test_capi import ERR_UNSUPPORTED, _call


@pytest.fixture(autouse=True)
def _built():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libdash_hip.so is not built (run __graft_entry__.build())")
    if torch.cuda.is_available():
        pytest.skip("argument checks are exercised where no device is present")


def _caches(layers):
    """One cache for each number of layers, a layer's page 4 bytes in one piece."""
    n = len(layers)
    return n, (ctypes.c_void_p * n)(*[0x100000] * n), (ctypes.c_int64 * (8 * n))(
        *[x for k in layers for x in (k, 64, 4, 1, 4, 1, 0, 4)])


def test_page_copies_of_too_many_tasks():
    lib = _lib.load()
    at = 0x100000
    for layers in ([16777216], [2 ** 31 - 1], [1] * 40 + [16777216], [1] * 70 + [9000000] * 2):
        n, base, desc = _caches(layers)
        assert lib.dash_copy_pages(n, base, desc, at, at, 3, 9, None) == ERR_UNSUPPORTED, layers
    for layers in ([67108864], [1] * 40 + [70000000]):
        n, base, desc = _caches(layers)
        assert lib.dash_keep_rows(n, base, desc, at, 4, at, at, at, 4, 2, 4, 8, 9, 4, None) == \
            ERR_UNSUPPORTED, layers
