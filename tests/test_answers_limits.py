"""Sizes that the operators of a step of several answers cannot launch are refused before any launch.  No GPU
calls."""

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


def test_rope_of_too_many_heads_or_tokens():
    rope = dict(q_sb=0, q_st=0, q_sh=128, qo_sb=0, qo_st=0, qo_sh=128, k_sb=0, k_st=0, k_sh=128, ko_sb=0, ko_st=0,
                ko_sh=128, dtype=1, positions_int64=0, pos_sb=0, pos_st=1, pairs=64, start=0, interleaved=0, back=0,
                factor=1.0, D=128, stream=None)
    append = dict(q_st=0, q_sh=128, qo_st=0, qo_sh=128, k_st=0, k_sh=128, v_st=0, v_sh=128, dtype=1,
                  positions_int64=0, kc_sp=128, kc_st=128, kc_sh=128, vc_sp=128, vc_st=128, vc_sh=128, page_size=16,
                  num_pages=9, pairs=64, start=0, interleaved=0, factor=1.0, D=128, stream=None)
    for H, Hkv in ((2 ** 27, 2 ** 27), (2 ** 26, 1), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1)):
        assert _call("dash_rope", **rope, H=H, Hkv=Hkv, B=1, S=5) == ERR_UNSUPPORTED, (H, Hkv)
        assert _call("dash_rope_append", **append, H=H, Hkv=Hkv, T=5) == ERR_UNSUPPORTED, (H, Hkv)
    # heads of 256 elements, 16 units of two chunks each: 2^32 units of a token, which is 0 in 32 bits
    assert _call("dash_rope_append", **{**append, "D": 256}, H=2 ** 27, Hkv=2 ** 26, T=5) == ERR_UNSUPPORTED
    assert _call("dash_rope", **rope, H=1, Hkv=1, B=2 ** 20, S=2 ** 20) == ERR_UNSUPPORTED
