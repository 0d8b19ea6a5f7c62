"""Workspace sizes of the attention of shared prompts: of sizes that no call takes, none is given.  No GPU calls."""

import ctypes

import pytest

from ananta_ocr_amd import _lib
from test_capi import ERR_UNSUPPORTED


@pytest.mark.parametrize("T, H, Hkv", [(2 ** 31 - 1, 2 ** 31 - 1, 1), (2 ** 30, 2 ** 10, 2 ** 10), (2 ** 25, 64, 8),
                                       (2 ** 31 - 1, 1, 1), (2 ** 26 - 3, 1, 1), (2 ** 29, 4, 4), (1, 2 ** 25, 2 ** 25)])
def test_sizes_that_are_refused(T, H, Hkv):
    nbytes = ctypes.c_int64(-7)
    assert _lib.load().dash_attn_shared_workspace_size(2, 1, H, Hkv, T, nbytes) == ERR_UNSUPPORTED
    assert nbytes.value == -7


@pytest.mark.parametrize("T, H, Hkv", [(2 ** 20 - 1, 64, 8), (2 ** 26 - 4, 1, 1), (0, 4, 4), (5, 4, 2)])
def test_sizes_that_are_taken(T, H, Hkv):
    nbytes = ctypes.c_int64(-7)
    assert _lib.load().dash_attn_shared_workspace_size(2, 1, H, Hkv, T, nbytes) == 0
    assert nbytes.value >= 2 * T * H * (128 * 4 + 8) + 8 * T
