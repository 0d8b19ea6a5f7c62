"""Sizes that the operators of a step of several answers cannot launch are refused before any launch.  No GPU
calls."""

import ctypes
import os

import pytest
import torch

from ananta_ocr_amd import _lib, sampling, shared_prefix
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


def test_shared_prompts_of_too_many_keys_or_rows():
    attn = dict(q_st=512, q_sh=128, k_sp=8192, k_sh=128, k_st=512, v_sp=8192, v_sh=128, v_st=512, table_stride=4, P=4,
                page_size=16, num_pages=9, out_bf16=0, o_st=512, o_sh=128, lse_st=4, lse_sh=1, B=2, G=1, H=4, Hkv=4,
                T=5, D=128, scale=0.1, workspace_bytes=1 << 60, stream=None)
    # keys whose tiles would end past 32 bits; rows, heads, sequences
    for kw in (dict(P=2 ** 27, page_size=16), dict(P=1, page_size=2 ** 31 - 127), dict(T=2 ** 31), dict(T=2 ** 40),
               dict(T=2 ** 29, H=2, Hkv=2), dict(T=1, H=2 ** 25, Hkv=2 ** 25), dict(B=8193), dict(G=8193)):
        assert _call("dash_attn_shared", **{**attn, **kw}) == ERR_UNSUPPORTED, kw
    for kw in (dict(T=2 ** 31), dict(T=2 ** 62), dict(B=8193), dict(G=8193)):
        size = {**dict(B=2, G=1, H=4, Hkv=4, T=5), **kw}
        assert _lib.load().dash_attn_shared_workspace_size(*size.values(), ctypes.c_int64()) == ERR_UNSUPPORTED, kw


def test_sampling_of_too_many_rows_or_tokens():
    sample = dict(row_stride=64, dtype=0, temperature0=1.0, top_k0=0, top_p0=1.0, min_p0=0.0, R=3, V=64,
                  probs_stride=64, probs_dtype=0, workspace_bytes=1 << 60, stream=None)
    for kw in (dict(R=2 ** 22), dict(R=2 ** 40), dict(V=2 ** 20 + 1)):
        assert _call("dash_sample", **{**sample, **kw}) == ERR_UNSUPPORTED, kw
    assert _lib.load().dash_sample_workspace_size(3, 2 ** 20 + 1, ctypes.c_int64()) == ERR_UNSUPPORTED


def test_inference_alone():
    """Calls whose gradients would be lost are refused."""
    q, k = torch.zeros(3, 4, 128, requires_grad=True), torch.zeros(5, 16, 2, 128)
    i = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="gradients"):
        shared_prefix.attn_shared(q, k, k, torch.zeros(2, 3, **i), torch.zeros(2, **i), torch.tensor([0, 1, 3], **i),
                                  None, None, 0.1)
    x = torch.zeros(2, 7, requires_grad=True)
    with pytest.raises(ValueError, match="gradients"):
        sampling.token_probs(x)
    with pytest.raises(ValueError, match="gradients"):
        sampling.sample(x, torch.zeros(2), return_probs=True)
