"""Trees of drafted tokens on the HIP kernels: their masks, the attention of their rows over a
cache, and the verification of the drafted tokens against the target's probabilities.

The nodes of the sequences are packed: rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 are the
nodes of sequence b, node 0 its root (the newest sampled token, whose key and value are not
committed yet), and ``parents`` holds each node's parent within its sequence, an earlier node.
The key and value of node i are written to the cache at slot context_len + i before the
attention.  max_query_len is at least the largest tree; rows that no tree has (a batch padded to a
fixed size) come out with nothing in particular, and prefix sums past the rows are cut to them.  ``pipeline.tree_step`` and
``pipeline.commit_tree`` are the whole step.

Like the other wrappers these take tensors of one GPU, allocate their outputs with torch, call one
C entry point on the current stream, and synchronise nothing.
"""

import contextlib
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _bf16_rows, _i32, _need_gpu, _ptr, _stream, _u8

MAX_NODES = 256                          # nodes of a sequence


_HERE = contextlib.nullcontext()


def _device(*ts):
    """A context in which the tensors' device is the current one (they must share it)."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            _need_gpu(*ts)
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    if index < 0:
        _need_gpu(*ts)
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _derivatives(*ts):
    """Whether a gradient of a tensor is asked for, or it carries a tangent (forward mode)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        return True
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _shape(t, shape, what):
    if t is not None and t.shape != shape:
        raise ValueError(f"{what}: {tuple(t.shape)} given, {tuple(shape)} needed")


def _nodes(cu_seqlens_q, max_query_len):
    n = int(max_query_len)
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() < 1:
        raise ValueError("cu_seqlens_q: [B + 1] needed")
    if n > MAX_NODES:
        raise NotImplementedError(f"trees of at most {MAX_NODES} nodes, got {n}")
    return cu_seqlens_q.numel() - 1, n


def tree_masks(parents, cu_seqlens_q, max_query_len):
    """(mask int64 [T, ceil(max_query_len / 64)], depth int32 [T]) of packed trees: bit m of a
    row's mask is set where node m of its sequence is the row's node or one of its ancestors;
    depth counts the ancestors.  parents [T] (within the sequence; -1, or a number that is not an
    earlier node's: none)."""
    B, n = _nodes(cu_seqlens_q, max_query_len)
    with _device(parents, cu_seqlens_q):
        par, cu = _i32(parents), _i32(cu_seqlens_q)
        T, words = par.numel(), (n + 63) // 64
        mask = torch.empty(T, words, dtype=torch.int64, device=par.device)
        depth = torch.empty(T, dtype=torch.int32, device=par.device)
        _lib.check(_lib.load().dash_tree_masks(_ptr(par), _ptr(cu), B, T, n, words, _ptr(mask),
                                               _ptr(depth), _stream()), "dash_tree_masks")
    return mask, depth


def tree_scores(idx_q, cu_seqlens_q, context_lens, depth, block_table, pool, block_size,
                local_blocks, max_query_len):
    """Router inputs of a tree's rows (dash_tree_scores): the block scores z [T, P] of idx_q
    [T, 128] fp32 against the k_bar pool's summaries of their sequences' committed blocks, the
    rows' positions (context_len + depth) and block counts [T] int32."""
    B, n = _nodes(cu_seqlens_q, max_query_len)
    T, d = idx_q.shape
    _shape(depth, (T,), "depth")
    _shape(context_lens, (B,), "context_lens")
    P = block_table.shape[1]
    _shape(block_table, (B, P), "block_table")
    _shape(pool, (pool.shape[0], d), "pool")
    if idx_q.dtype != torch.float32 or idx_q.stride(1) != 1 or pool.dtype != torch.float32 \
            or not pool.is_contiguous():
        raise ValueError("idx_q and the k_bar pool: contiguous fp32 rows are needed")
    with _device(idx_q, cu_seqlens_q, context_lens, depth, block_table, pool):
        cu, ctx, dep, bt = _i32(cu_seqlens_q), _i32(context_lens), _i32(depth), _i32(block_table)
        zs = max(32, (P + 31) // 32 * 32)
        z = torch.empty(T, zs, dtype=torch.float32, device=idx_q.device)
        rows = torch.empty(2, T, dtype=torch.int32, device=idx_q.device)
        _lib.check(_lib.load().dash_tree_scores(
            _ptr(idx_q), idx_q.stride(0), _ptr(cu), _ptr(ctx), _ptr(dep), _ptr(bt), bt.stride(0),
            _ptr(pool), pool.shape[0], B, T, n, P, d, int(block_size), int(local_blocks),
            _ptr(rows[0]), _ptr(rows[1]), _ptr(z), zs, _stream()), "dash_tree_scores")
    return z[:, :P], rows[0], rows[1]


def attn_tree(q, k, v, idx, bias, valid, mask, depth, context_lens, cu_seqlens_q, max_query_len,
              block_size, local_window, scale, block_table=None, page_size=None,
              out_dtype=torch.float32, return_lse=False):
    """Attention of a tree's rows q [T,H,128] over a cache with Hkv heads (H a multiple of Hkv):
    k/v pages [pages, page_size, Hkv, 128] with block_table [B,P], or contiguous [B,Hkv,S,128].
    Row r of sequence b, at position t = context_lens[b] + depth[r], attends

    * the committed keys (slots below context_lens[b]) of its window (t - local_window, t];
    * the committed keys below the window of its routed blocks idx [T,K] (valid, a block's first
      slot), with the bias of the slot;
    * the drafted keys (slot context_lens[b] + m) whose bit m is set in mask [T, words].

    idx, bias and valid may be None (no routed blocks).  block_size is 32 or a multiple of 64, at
    most 2,048 blocks a sequence and 64 slots a row.  Returns out [T,H,128] (fp32 or bf16) and
    with return_lse the log-sum-exp [T,H] fp32; a row that sees no key gives 0 and -inf."""
    lib = _lib.load()
    B, n = _nodes(cu_seqlens_q, max_query_len)
    q_shape, k_shape = q.shape, k.shape           # (a tensor's shape costs the host 0.2 us)
    if len(q_shape) != 3 or len(k_shape) != 4 or k_shape != v.shape:
        raise ValueError("q [T,H,D] and k, v of one shape [.., .., .., D] are needed")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise NotImplementedError("attn_tree writes fp32 or bf16")
    T, H, D = q_shape
    paged = block_table is not None
    Hkv = k_shape[2] if paged else k_shape[1]
    if k_shape[3] != D or Hkv == 0 or H % Hkv:
        raise ValueError(f"{H} query heads of {D} over {Hkv} key heads of {k_shape[3]}")
    K = 0 if idx is None else idx.shape[-1]
    if K:
        if bias is None:
            raise ValueError("routed blocks need their bias")
        _shape(idx, (T, K), "idx")
        _shape(bias, (T, K), "bias")
        _shape(valid, (T, K), "valid")
    _shape(depth, (T,), "depth")
    _shape(context_lens, (B,), "context_lens")
    _shape(mask, (T, (n + 63) // 64), "mask")
    if mask.dtype != torch.int64:
        raise ValueError("mask: int64 words")
    if paged:
        if block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError(f"block_table: {B} rows needed")
        if int(page_size or 0) != k_shape[1]:
            raise ValueError(f"page_size {page_size}: the pages hold {k_shape[1]} tokens")
        if block_table.shape[1] * k_shape[1] > 2 ** 31 - 1:
            raise NotImplementedError("a block_table of at most 2^31 - 1 tokens a sequence")
    elif k_shape[0] != B:
        raise ValueError(f"cache of {k_shape[0]} sequences, {B} trees")
    with _device(q, k, v, idx, bias, valid, mask, depth, context_lens, cu_seqlens_q, block_table):
        q, k, v = _bf16_rows(q), _bf16_rows(k), _bf16_rows(v)
        cu, ctx, dep, bt = _i32(cu_seqlens_q), _i32(context_lens), _i32(depth), _i32(block_table)
        mask = mask.contiguous()
        idx_c = bias_c = valid_c = None
        if K:
            idx_c, valid_c = _i32(idx), _u8(valid)
            bias_c = bias if bias.dtype == torch.float32 and bias.is_contiguous() \
                else bias.float().contiguous()
        out = torch.empty(T, H, D, dtype=out_dtype, device=q.device)
        lse = torch.empty(T, H, dtype=torch.float32, device=q.device) if return_lse else None
        if T:
            qs, (ks, k1, k2, _), (vs, v1, v2, _) = q.stride(), k.stride(), v.stride()
            if paged:
                S, pages, bt_stride = bt.shape[1] * k_shape[1], k_shape[0], bt.stride(0)
                kh, kt, vh, vt = k2, k1, v2, v1
            else:
                S, pages, bt_stride = k_shape[2], 0, 0
                kh, kt, vh, vt = k1, k2, v1, v2
            lw = min(int(local_window), 1 << 30)      # (past every position it is the same window)
            nbytes = _attn_workspace(B, H, Hkv, T, n, K, S, int(block_size), lw)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            _lib.check(lib.dash_attn_tree(
                q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks, kh, kt, v.data_ptr(), vs, vh, vt,
                _ptr(bt), bt_stride, int(page_size or 0), pages,
                ctx.data_ptr(), cu.data_ptr(), _ptr(idx_c), _ptr(valid_c), _ptr(bias_c), K,
                mask.data_ptr(), (n + 63) // 64, dep.data_ptr(), out.data_ptr(),
                int(out_dtype == torch.bfloat16), H * D, D, _ptr(lse),
                0 if lse is None else H, 1, B, H, Hkv, T, n, S, D, int(block_size),
                lw, float(scale), _ptr(ws), nbytes, _stream()),
                "dash_attn_tree")
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _attn_workspace(*sizes):
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().dash_attn_tree_workspace_size(*sizes, nbytes), "workspace")
    return nbytes.value


@functools.lru_cache(maxsize=256)
def _verify_workspace(*sizes):
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().dash_verify_tree_workspace_size(*sizes, nbytes), "workspace")
    return max(nbytes.value, 256)


_VERIFY_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def verify_tree(target, tokens, parents, cu_seqlens_q, max_query_len, uniforms=None, draft=None):
    """Which drafted tokens stand: (count int32 [B], path int32 [B, max_query_len], next_token
    int64 [B]).  target [T,V]: row r holds the target's probabilities of the token after node r
    (greedy: any scores); tokens [T] the nodes' tokens (the root's is not read).

    * uniforms None: greedy.  The path follows, from the root on, the child whose token is its
      parent's best one (the lowest id of equals), and next_token is the last node's.
    * uniforms [T], draft None: children are certain proposals (a draft's best tokens).  With Z = 1
      child x is accepted if its uniform times Z is below p(x); else x leaves p, and Z -= p(x).
    * uniforms [T] and draft [T,V] (row r: the probabilities node r's children were drawn from,
      each by itself): with a = 0 and Z = 1 accepted if u Z q(x) < max(p(x) - a q(x), 0); else
      a += Z and Z = sum(max(p - a q, 0)).

    The uniform of the root draws next_token from what is left at the last accepted node: the first
    id whose running sum exceeds it times the whole.  Uniforms lie in [0, 1); probabilities and
    uniforms that are not above 0 (NaN too) count as 0.  path holds the accepted nodes, the root
    first, then -1; a sequence without nodes has count 0 and next_token -1.  The three are views of one
    allocation with the call's workspace (some KB; greedy 8 B a row and piece of it): clone what is
    kept for long or saved."""
    lib = _lib.load()
    B, n = _nodes(cu_seqlens_q, max_query_len)
    if target.dim() != 2 or target.shape[1] == 0:
        raise ValueError("target: [T, V] needed")
    T, V = target.shape
    for t, what in ((tokens, "tokens"), (parents, "parents"), (uniforms, "uniforms")):
        _shape(t, (T,), what)
    _shape(draft, (T, V), "draft")
    if draft is not None and uniforms is None:
        raise ValueError("draft probabilities need uniforms")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("tokens: int32 or int64")
    with _device(target, tokens, parents, cu_seqlens_q, uniforms, draft):
        if target.dtype not in _VERIFY_TYPES or (draft is not None and draft.dtype != target.dtype):
            target = target.float()
            draft = None if draft is None else draft.float()
        if target.stride(1) != 1:
            target = target.contiguous()
        if draft is not None and draft.stride(1) != 1:
            draft = draft.contiguous()
        tok, par, cu = tokens.contiguous(), _i32(parents), _i32(cu_seqlens_q)
        u = None if uniforms is None else uniforms.float().contiguous()
        # outputs and workspace (some KB) of one allocation: 1.5 us less than four
        words = _verify_workspace(B, T, V, int(u is None)) // 4
        sizes = (words, 2 * B, B, B * n)
        ws, token, count, path = torch.empty(sum(sizes), dtype=torch.int32,
                                             device=target.device).split_with_sizes(sizes)
        token, path = token.view(torch.int64), path.view(B, n)
        _lib.check(lib.dash_verify_tree(
            _ptr(target), target.stride(0), _ptr(draft), 0 if draft is None else draft.stride(0),
            _VERIFY_TYPES[target.dtype], _ptr(tok), int(tok.dtype == torch.int64), _ptr(par),
            _ptr(cu), _ptr(u), B, T, V, n, _ptr(count), _ptr(path), path.stride(0), _ptr(token),
            _ptr(ws), 4 * words, _stream()), "dash_verify_tree")
    return count, path, token
