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


def test_launches_of_too_many_work_groups():
    ver = dict(target_stride=9, draft_stride=9, dtype=0, tokens_int64=1, B=2, V=9, max_query_len=4,
               path_stride=4, workspace_bytes=1 << 60, uniforms=None, draft=None, stream=None)
    for T in (16777216, 2 ** 31, 2 ** 40):
        assert _call("dash_verify_tree", **{**ver, "T": T}) == ERR_UNSUPPORTED, T
    attn = dict(q_st=512, q_sh=128, k_sb=0, k_sh=128, k_st=256, v_sb=0, v_sh=128, v_st=256,
                table_stride=4, page_size=64, num_pages=9, K=3, words=1, out_bf16=0, o_st=512,
                o_sh=128, lse_st=4, lse_sh=1, H=4, Hkv=4, max_query_len=4, S=256, D=128,
                block_size=64, local_window=128, scale=0.1, workspace_bytes=1 << 60, stream=None)
    # one work-group a (sequence, key head); several, whose sums are added up; rows past 32 bits
    for kw in (dict(B=8388608, T=16), dict(B=2, T=16777217), dict(B=2, T=2 ** 31, H=1, Hkv=1)):
        assert _call("dash_attn_tree", **{**attn, **kw}) == ERR_UNSUPPORTED, kw
    assert _call("dash_tree_masks", B=16777216, T=5, max_query_len=4, words=1, stream=None) == \
        ERR_UNSUPPORTED
    state = dict(num_pages=9, table_stride=4, P=4, page_size=8, stream=None)
    for name in ("dash_free_pages", "dash_compact_pages"):
        assert _call(name, **{**state, "R": 8193}) == ERR_UNSUPPORTED, name
    assert _call("dash_compact_pages", **{**state, "R": 8192, "P": 600000}) == ERR_UNSUPPORTED
    scores = dict(iq_st=128, table_stride=4, pool_rows=9, B=2, T=5, max_query_len=4, nblk=4, d=128,
                  block_size=64, local_blocks=2, z_stride=32, stream=None)
    for kw in (dict(max_query_len=257), dict(max_query_len=2 ** 31 - 1), dict(nblk=2 ** 22), dict(B=65536),
               dict(T=2 ** 31 - 1)):
        assert _call("dash_tree_scores", **{**scores, **kw}) == ERR_UNSUPPORTED, kw
    kbar = dict(ik_st=128, ik_sp=8192, table_stride=4, pool_rows=9, B=2, nblk=4, d=128, block_size=64,
                stream=None)
    for kw in (dict(nblk=16777216, block_size=1), dict(nblk=2 ** 26), dict(B=65536)):
        assert _call("dash_kbar_pages", **{**kbar, **kw}) == ERR_UNSUPPORTED, kw


def test_tables_whose_wanted_pages_pass_32_bits():
    """8,192 rows that each want 262,144 pages or more would add up to a number below 0."""
    state = dict(num_pages=9, table_stride=1 << 18, R=8192, page_size=8, stream=None)
    assert _call("dash_reserve_pages", **{**state, "P": 1 << 18}) == ERR_UNSUPPORTED
    assert _call("dash_reserve_pages", **{**state, "R": 3, "P": 2 ** 31 - 1}) == ERR_UNSUPPORTED
