"""What trees, verification and page calls refuse on the host: shapes, types, limits, host memory.
No GPU calls."""

import os

import pytest
import torch

from ananta_ocr_amd import _lib, kv_pages, ops, pipeline, tree
from test_capi import ERR_INVALID, ERR_UNSUPPORTED, _call
from tree_oracle import Pages, ancestors, verify

I32 = torch.int32


def _attn(**kw):
    T, B, n = 5, 2, 4
    a = dict(q=torch.zeros(T, 4, 128), k=torch.zeros(3, 64, 2, 128), v=torch.zeros(3, 64, 2, 128),
             idx=torch.zeros(T, 3, dtype=I32), bias=torch.zeros(T, 3), valid=None,
             mask=torch.zeros(T, 1, dtype=torch.int64), depth=torch.zeros(T, dtype=I32),
             context_lens=torch.zeros(B, dtype=I32), cu_seqlens_q=torch.tensor([0, 1, 5]),
             max_query_len=n, block_size=64, local_window=128, scale=0.1,
             block_table=torch.zeros(B, 2, dtype=I32), page_size=64)
    a.update(kw)
    return tree.attn_tree(**a)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(5, 3, 128)), dict(q=torch.zeros(5, 512)), dict(v=torch.zeros(3, 64, 2, 64)),
    dict(idx=torch.zeros(4, 3)), dict(bias=torch.zeros(5, 2)), dict(valid=torch.zeros(5, 2)),
    dict(bias=None), dict(mask=torch.zeros(5, 2, dtype=torch.int64)),
    dict(mask=torch.zeros(5, 1, dtype=I32)), dict(depth=torch.zeros(4)),
    dict(context_lens=torch.zeros(3)), dict(block_table=torch.zeros(3, 2, dtype=I32)),
    dict(page_size=128), dict(page_size=None), dict(cu_seqlens_q=torch.zeros(2, 2)),
    dict(block_table=None, page_size=None)])
def test_attn_tree_refuses_shapes(kw):
    with pytest.raises(ValueError):
        _attn(**kw)


def test_attn_tree_refuses_sizes_types_and_host_memory():
    with pytest.raises(NotImplementedError):
        _attn(max_query_len=257)
    with pytest.raises(NotImplementedError):
        _attn(out_dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        _attn()
    with pytest.raises(ValueError, match="GPU"):
        tree.tree_masks(torch.zeros(3), torch.tensor([0, 3]), 3)
    with pytest.raises(NotImplementedError):
        tree.tree_masks(torch.zeros(3), torch.tensor([0, 3]), 1000)
    with pytest.raises(NotImplementedError):
        pipeline.tree_step(pipeline.DecodeState(None), *[None] * 16)


@pytest.mark.parametrize("kw", [
    dict(target=torch.zeros(5)), dict(target=torch.zeros(5, 0)), dict(tokens=torch.zeros(4).long()),
    dict(tokens=torch.zeros(5)), dict(parents=torch.zeros(6)), dict(uniforms=torch.zeros(4)),
    dict(draft=torch.zeros(5, 8)), dict(draft=torch.zeros(5, 9), uniforms=None)])
def test_verify_refuses(kw):
    a = dict(target=torch.zeros(5, 9), tokens=torch.zeros(5).long(), parents=torch.zeros(5),
             cu_seqlens_q=torch.tensor([0, 5]), max_query_len=5, uniforms=torch.zeros(5), draft=None)
    with pytest.raises(ValueError, match="GPU"):
        tree.verify_tree(**a)
    with pytest.raises(ValueError) as e:
        tree.verify_tree(**{**a, **kw})
    assert "GPU" not in str(e.value)


def test_scores_and_summaries_refuse():
    a = dict(idx_q=torch.zeros(5, 128), cu_seqlens_q=torch.tensor([0, 5]), context_lens=torch.zeros(1, dtype=I32),
             depth=torch.zeros(5, dtype=I32), block_table=torch.zeros(1, 2, dtype=I32),
             pool=torch.zeros(3, 128), block_size=64, local_blocks=2, max_query_len=5)
    b = dict(idx_k=torch.zeros(3, 64, 128), head_cls=torch.zeros(128), first_tokens=torch.zeros(1, dtype=I32),
             seq_lens=torch.zeros(1, dtype=I32), block_table=torch.zeros(1, 2, dtype=I32),
             pool=torch.zeros(3, 128), block_size=64)
    for f, good, bad in (
            (tree.tree_scores, a, [dict(idx_q=a["idx_q"].half()), dict(pool=a["pool"].half()),
                                   dict(pool=torch.zeros(3, 64)), dict(pool=torch.zeros(3, 256)[:, :128]),
                                   dict(block_table=torch.zeros(2, 2, dtype=I32)), dict(depth=torch.zeros(4))]),
            (ops.kbar_pages, b, [dict(idx_k=torch.zeros(2, 64, 128)), dict(pool=torch.zeros(3, 64)),
                                 dict(idx_k=torch.zeros(3, 64, 128).half()), dict(head_cls=torch.zeros(64)),
                                 dict(seq_lens=torch.zeros(2)), dict(block_size=32)])):
        with pytest.raises(ValueError, match="GPU"):
            f(**good)
        for kw in bad:
            with pytest.raises((ValueError, NotImplementedError)) as e:
                f(**{**good, **kw})
            assert "GPU" not in str(e.value)


def test_page_calls_refuse():
    refs, table, lens = torch.zeros(9, dtype=I32), torch.zeros(3, 4, dtype=I32), torch.zeros(3, dtype=I32)
    rows = torch.zeros(2, dtype=I32)
    for f, more in ((kv_pages.fork_pages, (rows, rows)), (kv_pages.reserve_pages, (lens,)),
                    (kv_pages.free_pages, (lens,)), (kv_pages.compact_pages, ())):
        with pytest.raises(ValueError, match="GPU"):
            f(refs, table, lens, *more, 8)
        for bad in ((refs[:0], table, lens), (refs, lens, lens), (refs, table, rows)):
            with pytest.raises(ValueError) as e:
                f(*bad, *more, 8)
            assert "GPU" not in str(e.value)
        with pytest.raises(ValueError, match="page_size"):
            f(refs, table, lens, *more, 0)
        big = torch.zeros(8193, 1, dtype=I32)
        with pytest.raises(NotImplementedError):
            f(refs, big, big[:, 0].contiguous(), *((big[:, 0].contiguous(),) * len(more)), 8)
        if more:
            with pytest.raises(ValueError, match="int32"):
                f(refs.long(), table, lens, *more, 8)
            with pytest.raises(ValueError, match="int32"):
                f(refs, table.t().contiguous().t(), lens, *more, 8)
    with pytest.raises(ValueError, match="dst"):
        kv_pages.fork_pages(refs, table, lens, rows, lens, 8)
    with pytest.raises(ValueError, match="new_lens"):
        kv_pages.reserve_pages(refs, table, lens, rows, 8)
    with pytest.raises(ValueError, match="GPU"):
        kv_pages.PageCaches([torch.zeros(4, 8, 2)])
    with pytest.raises(ValueError):
        kv_pages.PageCaches([])
    with pytest.raises(ValueError):
        kv_pages.PageCaches([], pages=[torch.zeros(4, 2)])


def _built():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libdash_hip.so is not built (run __graft_entry__.build())")
    if torch.cuda.is_available():
        pytest.skip("argument checks are exercised where no device is present")


def test_entry_points_check_before_any_device_call():
    """Sizes past a kernel's limits and missing arguments return before a launch."""
    _built()
    attn = dict(q_st=512, q_sh=128, k_sb=0, k_sh=128, k_st=256, v_sb=0, v_sh=128, v_st=256,
                table_stride=4, page_size=64, num_pages=9, K=3, words=1, out_bf16=0, o_st=512,
                o_sh=128, lse_st=4, lse_sh=1, B=2, H=4, Hkv=2, T=5, max_query_len=4, S=256, D=128,
                block_size=64, local_window=128, scale=0.1, workspace_bytes=1 << 40, stream=None)
    for kw, want in ((dict(D=64), ERR_UNSUPPORTED), (dict(Hkv=3), ERR_UNSUPPORTED),
                     (dict(K=65), ERR_UNSUPPORTED), (dict(max_query_len=257, words=5), ERR_UNSUPPORTED),
                     (dict(words=2), ERR_UNSUPPORTED), (dict(block_size=48), ERR_UNSUPPORTED),
                     (dict(page_size=96), ERR_UNSUPPORTED), (dict(page_size=0), ERR_UNSUPPORTED),
                     (dict(S=64 * 2049), ERR_UNSUPPORTED), (dict(k_st=4), ERR_UNSUPPORTED),
                     (dict(scale=0.0), ERR_UNSUPPORTED), (dict(num_pages=0), ERR_INVALID),
                     (dict(local_window=0), ERR_INVALID), (dict(mask=None), ERR_INVALID),
                     (dict(bias=None), ERR_INVALID), (dict(T=-1), ERR_INVALID)):
        assert _call("dash_attn_tree", **{**attn, **kw}) == want, kw
    assert _call("dash_attn_tree", **{**attn, "T": 0, "q": None}) == 0
    ver = dict(target_stride=9, draft_stride=9, dtype=0, tokens_int64=1, B=2, T=5, V=9,
               max_query_len=4, path_stride=4, workspace_bytes=1 << 40, stream=None)
    for kw, want in ((dict(dtype=3), ERR_INVALID), (dict(V=0), ERR_INVALID),
                     (dict(uniforms=None), ERR_INVALID), (dict(max_query_len=300), ERR_UNSUPPORTED),
                     (dict(B=70000), ERR_UNSUPPORTED), (dict(workspace_bytes=10), -4),
                     (dict(workspace=None), -4)):
        assert _call("dash_verify_tree", **{**ver, **kw}) == want, kw
    state = dict(num_pages=9, table_stride=4, R=3, P=4, page_size=8, stream=None)
    for name, more in (("dash_fork_pages", dict(n=2)), ("dash_reserve_pages", {}),
                       ("dash_free_pages", {}), ("dash_compact_pages", {})):
        for kw, want in ((dict(page_size=0), ERR_INVALID), (dict(R=-1), ERR_INVALID),
                         (dict(refs=None), ERR_INVALID), (dict(lens=None), ERR_INVALID)):
            assert _call(name, **{**state, **more, **kw}) == want, (name, kw)
    for name in ("dash_fork_pages", "dash_reserve_pages"):
        assert _call(name, **{**state, "n": 2, "R": 8193}) == ERR_UNSUPPORTED
    assert _call("dash_copy_pages", num_caches=1, num_pairs=1, num_pages=1, stream=None,
                 from_pages=None) == ERR_INVALID
    assert _call("dash_copy_pages", num_caches=1, num_pairs=0, num_pages=1, stream=None) == 0
    masks = dict(B=2, T=5, max_query_len=4, words=1, stream=None)
    assert _call("dash_tree_masks", **{**masks, "words": 2}) == ERR_UNSUPPORTED
    assert _call("dash_tree_masks", **{**masks, "max_query_len": 999, "words": 16}) == ERR_UNSUPPORTED
    assert _call("dash_tree_masks", **{**masks, "parents": None}) == ERR_INVALID


def test_oracle_by_hand():
    assert ancestors([-1, 0, 0, 1], 3) == [3, 1, 0]
    p = torch.tensor([[0.5, 0.3, 0.2], [0.0, 0.0, 1.0], [0.1, 0.8, 0.1]])
    # child 1 (token 1): 0.29 < 0.3 accepted; its child none; drawn from row 1
    assert verify(p, [0, 1, 0], [-1, 0, 0], torch.tensor([0.4, 0.29, 0.9])) == ([0, 1], 2)
    # 0.31 rejected, then token 0: 0.9 * 0.7 >= 0.5 rejected: token 2 is left
    assert verify(p, [0, 1, 0], [-1, 0, 0], torch.tensor([0.4, 0.31, 0.9])) == ([0], 2)
    # with draft probabilities: 0.5 * 0.6 >= 0.3, left (0.4, 0, 0): token 0
    q = torch.tensor([[0.1, 0.6, 0.3]] * 3)
    assert verify(p, [0, 1, 1], [-1, 0, 0], torch.tensor([0.4, 0.5, 0.9]), q) == ([0], 0)
    assert verify(p, [0, 0, 2], [-1, 0, 1]) == ([0, 1, 2], 1)
    a = Pages(4, 3, 4, 8)
    assert a.reserve([9, 0, 0])[0] == 1 and a.fork([0], [2]) == (1, [1], [2])
    assert a.refs == [2, 1, 1, 0] and a.table[2][:2] == [0, 2]
    a.free([0, 0, 9])
    assert a.refs == [1, 0, 1, 0] and a.compact() == ([2], [1]) and a.table[2][:2] == [0, 1]


def _addresses(desc, i, rows):
    """Byte offsets of a layer's page (or row) of cache i, as the kernels walk its descriptor."""
    _, _, _, n1, s1, n2, s2, seg = desc[8 * i:8 * i + 8]
    return sorted(a * s1 + b * s2 + x for a in range(1 if rows else n1) for b in range(n2)
                  for x in range(seg))


@pytest.mark.parametrize("make", [
    lambda: torch.zeros(2, 5, 4, 3, 8), lambda: torch.zeros(2, 5, 3, 4, 8).transpose(2, 3),
    lambda: torch.zeros(2, 5, 2, 4, 3, 8)[:, :, 1], lambda: torch.zeros(2, 5, 4, 3, 10)[..., 1:9],
    lambda: torch.zeros(2, 5, 4, 8, 3).transpose(3, 4), lambda: torch.zeros(2, 5, 4, 1, 8),
    lambda: torch.zeros(5, 2, 4, 3, 8).transpose(0, 1), lambda: torch.zeros(2, 5, 4),
    lambda: torch.zeros(2, 5, 4, 3, 8, dtype=torch.int8),
    lambda: torch.zeros(2, 1, 5, 8).transpose(1, 2), lambda: torch.zeros(2, 5, 1, 4, 8).transpose(2, 3)])
def test_descriptors_cover_a_page_and_a_row(make):
    t = make()
    es = t.element_size()
    offs = torch.zeros(t.shape[1:], dtype=torch.int64)
    for a, (n, st) in enumerate(zip(t.shape[1:], t.stride()[1:])):
        offs += (torch.arange(n) * st).view(*[-1 if b == a else 1 for b in range(offs.dim())])
    n, base, desc = kv_pages.PageCaches._describe([(t, 2)], 1)
    page = [x * es + y for x in offs[0].flatten().tolist() for y in range(es)]
    assert n == 1 and base[0] == t.data_ptr() and _addresses(desc, 0, False) == sorted(page)
    assert list(desc[0:3]) == [2, t.stride(0) * es, t.stride(1) * es]
    _, _, desc = kv_pages.PageCaches._describe([(t, 3)], 1)
    row = [x * es + y for x in offs[0, 0].flatten().tolist() for y in range(es)]
    assert _addresses(desc, 0, True) == sorted(row) and desc[4] == t.stride(2) * es


def test_descriptors_refuse_overlaps():
    for t in (torch.zeros(4, 1, 8).expand(4, 6, 8), torch.zeros(1, 6, 8).expand(4, 6, 8),
              torch.zeros(200).as_strided((4, 6, 8), (48, 5, 1))):
        with pytest.raises(ValueError, match="overlap"):
            kv_pages.PageCaches._describe([(t, 1)], 0)
