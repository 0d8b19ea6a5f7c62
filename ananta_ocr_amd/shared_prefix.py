"""Full attention of a batch whose sequences share prompts, on the HIP kernels (csrc/dash_shared.h): the
layers of a decoder that do not route, over a paged cache whose rows were forked
(kv_pages.PagePool.fork).  The keys of a shared prompt are read once for all of its answers.
"""

import ctypes
import functools

import torch

from . import _lib
from .ops import _i32, _ptr, _rows, _stream
from .tree import _derivatives, _device, _shape

MAX_SEQS = 8192
MAX_TOKENS = 2 ** 31 - 128


def _bf16(*ts):
    """Refuses other types: a cast would round queries, and copy a whole pool at every call."""
    if any(t.dtype != torch.bfloat16 for t in ts):
        raise NotImplementedError(f"queries and caches in bf16: {', '.join(str(t.dtype) for t in ts)}")


def attn_shared(q, k, v, block_table, context_lens, cu_seqlens_q, cu_groups, prefix_lens, scale,
                out_dtype=torch.float32, return_lse=False):
    """Attention of new tokens q [T,H,128] over pages k/v [pages, page_size, Hkv, 128] (bf16, H a
    multiple of Hkv, any page size) through block_table [B,P].  Rows cu_seqlens_q[b] ..
    cu_seqlens_q[b + 1] - 1 are the new tokens of sequence b, at positions context_lens[b] + i, their
    keys and values already written (rope.rope_append); each attends every key of its sequence up to
    itself.

    Sequences cu_groups[g] .. cu_groups[g + 1] - 1 (cu_groups [G + 1], prefix sums over the batch) have
    the keys below prefix_lens[g] in common: they are read through one table row, once for the group,
    that of the first sequence with new tokens that holds them all (or the most of them).  Sequences
    without new tokens, as an answer that has left, may hold anything.  A forked row shares its full
    pages, and a copy of the partly filled one holds the same keys.  Sequences of no group, or of one
    with a prefix of 0, share nothing; cu_groups and prefix_lens may be None.  Prefix sums past the
    rows or the batch are cut to them.

    Returns out [T,H,128] (fp32 or bf16) and with return_lse the log-sum-exp [T,H] fp32; a row that
    sees no key, or of no sequence (a batch padded to a fixed size), gives 0 and -inf.  At most 8,192
    sequences; 2^31 - 128 tokens a table row.  For inference: no gradients."""
    if q.dim() != 3 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q [T,H,D] and k, v of one shape [pages, page_size, Hkv, D] are needed")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise NotImplementedError("attn_shared writes fp32 or bf16")
    T, H, D = q.shape
    pages, page_size, Hkv = k.shape[:3]
    if k.shape[3] != D or Hkv == 0 or H % Hkv or page_size == 0:
        raise ValueError(f"{H} query heads of {D} over {Hkv} key heads of {k.shape[3]}, pages of {page_size}")
    if block_table.dim() != 2:
        raise ValueError("block_table [B, P] is needed")
    B, P = block_table.shape
    _shape(context_lens, (B,), "context_lens")
    _shape(cu_seqlens_q, (B + 1,), "cu_seqlens_q")
    if (cu_groups is None) != (prefix_lens is None):
        raise ValueError("cu_groups and prefix_lens go together")
    G = 0
    if cu_groups is not None:
        if cu_groups.dim() != 1 or cu_groups.numel() < 1:
            raise ValueError("cu_groups: [G + 1] needed")
        G = cu_groups.numel() - 1
        _shape(prefix_lens, (G,), "prefix_lens")
    if B > MAX_SEQS or G > MAX_SEQS:
        raise NotImplementedError(f"at most {MAX_SEQS} sequences and groups")
    if P * page_size > MAX_TOKENS:
        raise NotImplementedError("a block_table of at most 2^31 - 128 tokens a sequence")
    if _derivatives(q, k, v):
        raise ValueError("attn_shared has no gradients")
    with _device(q, k, v, block_table, context_lens, cu_seqlens_q, cu_groups, prefix_lens):
        _bf16(q, k, v)
        q, k, v = _rows(q), _rows(k), _rows(v)
        bt, ctx, cu = _i32(block_table), _i32(context_lens), _i32(cu_seqlens_q)
        gr, pre = _i32(cu_groups), _i32(prefix_lens)
        out = torch.empty(T, H, D, dtype=out_dtype, device=q.device)
        lse = torch.empty(T, H, dtype=torch.float32, device=q.device) if return_lse else None
        if T and H:
            nbytes = _workspace(B, G, H, Hkv, T)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            (qt, qh, _), (kp, kt, kh, _), (vp, vt, vh, _) = q.stride(), k.stride(), v.stride()
            _lib.check(_lib.load().dash_attn_shared(
                q.data_ptr(), qt, qh, _ptr(k), kp, kt, kh, _ptr(v), vp, vt, vh, _ptr(bt), bt.stride(0), P,
                page_size, pages, _ptr(ctx), _ptr(cu), _ptr(gr), _ptr(pre), out.data_ptr(),
                int(out_dtype == torch.bfloat16), H * D, D, _ptr(lse), H, 1, B, G, H, Hkv, T, D,
                float(scale), ws.data_ptr(), nbytes, _stream()), "dash_attn_shared")
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _workspace(*sizes):
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().dash_attn_shared_workspace_size(*sizes, nbytes), "workspace")
    return nbytes.value
