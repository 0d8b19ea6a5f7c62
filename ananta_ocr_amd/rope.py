"""Rotary positions on the HIP kernels (csrc/dash_rope.hip): queries and keys turned by their
positions, with a backward pass for training, or turned and written to a paged cache in one launch
for serving.

A part [start, start + 2 m) of every head row is turned, m = len(inv_freq): pair j is elements (j,
j + m) of the part, or (2 j, 2 j + 1) where ``interleaved``, its angle position * inv_freq[j].  Angles
are taken in 64 bits (a position of 10^5 is 10^5 radians, which 32 bits hold to 4e-3), their sines and
cosines to 1.2e-10 and rounded to 32 bits before the products, which are rounded once to the rows' type.

``inv_freq`` gives the frequencies of a head with the usual scalings for long contexts; the cos/sin
tables of two-axis positions are page_rope's.
"""

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _need_gpu, _ptr, _stream
from .tree import _derivatives, _device, _shape

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_PAIRS = 256


def inv_freq(dim, base=10000.0, scaling=None, device=None):
    """(frequencies [dim / 2] float64, factor) of a rotary part of `dim` elements: base^(-2 j / dim).
    scaling (None, or a configuration's rope_scaling) stretches them for long contexts:

    * {"type": "linear", "factor": s}: all divided by s;
    * {"type": "ntk", "factor": s}: the base times s^(dim / (dim - 2)), so that the lowest
      frequency is divided by s and the highest kept;
    * {"type": "yarn", "factor": s, "original_max_position_embeddings": n, "beta_fast": 32,
      "beta_slow": 1, "mscale": 1, "mscale_all_dim": 0}: frequencies of fewer than beta_slow turns
      over n positions are divided by s, those of more than beta_fast kept, with a linear ramp over
      the index between (from the whole index below to the one above, or with "truncate": False from
      the border itself); factor is "attention_factor" where that is given, else g(mscale) /
      g(mscale_all_dim), g(x) = 0.1 x ln s + 1 (1 where s <= 1).

    `factor` scales cos and sin (1 for the others, which refuse an "attention_factor" that is not).
    Other settings are not read."""
    dim = int(dim)
    if dim < 0 or dim % 2:
        raise ValueError(f"a rotary part of {dim} elements")
    m = dim // 2
    kind = None if scaling is None else scaling.get("type", scaling.get("rope_type", "default"))
    s = 1.0 if scaling is None else float(scaling.get("factor", 1.0))
    given = None if scaling is None else scaling.get("attention_factor")
    if not s > 0.0:
        raise ValueError(f"a scaling factor of {s}")
    base, factor = float(base), 1.0
    if kind == "ntk" and dim > 2:
        base *= s ** (dim / (dim - 2))
    f = base ** (-torch.arange(m, dtype=torch.float64) / max(m, 1))
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        n = float(scaling["original_max_position_embeddings"])

        def at(turns):                       # the index whose frequency makes so many turns
            return m * math.log(n / (turns * 2 * math.pi)) / math.log(base)

        lo, hi = at(float(scaling.get("beta_fast", 32))), at(float(scaling.get("beta_slow", 1)))
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, dim - 1)
        ramp = ((torch.arange(m, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / s * ramp + f * (1 - ramp)

        def g(x):
            return 0.1 * x * math.log(s) + 1.0 if s > 1 else 1.0

        if given is None:
            factor = g(float(scaling.get("mscale", 1))) / g(float(scaling.get("mscale_all_dim", 0)))
        else:
            factor = float(given)
    elif kind not in (None, "default", "ntk"):
        raise NotImplementedError(f"rope scaling {kind!r}")
    if kind != "yarn" and given is not None and float(given) != 1.0:
        raise NotImplementedError(f"rope scaling {kind!r} with an attention factor of {given}")
    return f if device is None else f.to(device), factor


def _freqs(inv_freq):
    if inv_freq.dim() != 1:
        raise ValueError("inv_freq: [pairs] needed")
    return inv_freq.to(torch.float64).contiguous()


def _part(D, m, start):
    if D % 2 or m > MAX_PAIRS:
        raise NotImplementedError(f"heads of an even width and at most {MAX_PAIRS} pairs: {D}, {m}")
    if start < 0 or start + 2 * m > D:
        raise ValueError(f"the part [{start}, {start + 2 * m}) of heads of {D}")


def _inner(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _leaves_in_capture(*xs):
    """Refuses a leaf, under capture, that an eager graph still refers to.  Its gradient is added up
    on the stream of that graph's forward: a backward pass captured now makes that stream part of the
    capture, which then ends the process.  A leaf's accumulating node lives as long as some graph
    refers to it; one that keeps what was noted on it, with no reference of ours left, is such a node,
    and one that was first seen in a capture on this stream is not."""
    if not torch._C._cuda_isCurrentStreamCapturing():
        return
    stream = _stream()
    for x in xs:
        if x is None or not x.requires_grad or not x.is_leaf:
            continue
        node = torch.autograd.graph.get_gradient_edge(x).node
        if node.metadata.get("dash_capture") == stream:
            continue
        node.metadata["dash_alive"] = True
        del node
        node = torch.autograd.graph.get_gradient_edge(x).node
        if node.metadata.pop("dash_alive", False):
            raise RuntimeError("apply_rope under capture: an eager graph of this leaf is still alive; "
                               "drop its outputs first, or pass x.detach().requires_grad_()")
        yield node                           # (kept by the caller until the graph refers to it)
        node.metadata["dash_capture"] = stream


class _RopeFn(torch.autograd.Function):
    """The turn by position * inv_freq (back: by the negative), times factor.  Its gradient is the
    turn the other way, so that this function is its own backward, to any order."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, interleaved, start, factor, back):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, freqs)
            ctx.shapes = q is not None and q.shape, k is not None and k.shape
        ctx.how = interleaved, start, factor, back
        return _turn(q, k, positions, freqs, interleaved, start, factor, back)

    @staticmethod
    def backward(ctx, dq, dk):
        interleaved, start, factor, back = ctx.how
        pos, freqs = ctx.saved_tensors
        if dq is not None or dk is not None:
            dq, dk = _rope(dq, dk, pos, freqs, interleaved, start, factor, not back)
        return dq, dk, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        pos, freqs = ctx.saved_tensors
        outs = _rope(tq, tk, pos, freqs, *ctx.how)
        some = tq if tq is not None else tk      # (the tangent of an output whose input has none is 0)
        return tuple(some.new_zeros(s) if y is None and s else y for s, y in zip(ctx.shapes, outs))


def _rope(q, k, *how):
    """_turn, recorded where a gradient or a tangent is."""
    if _derivatives(q, k):
        return _RopeFn.apply(q, k, *how)
    return _turn(q, k, *how)


def _turn(q, k, pos, freqs, interleaved, start, factor, back):
    args, outs = [], []
    for x in (q, k):
        if x is None:
            args += [None, 0, 0, 0, 0, None, 0, 0, 0]
            outs.append(None)
            continue
        x = _inner(x)
        y = torch.empty_like(x)
        if y.stride(-1) != 1 and y.shape[-1] != 1:
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        outs.append(y)
        lead = (0,) if x.dim() == 3 else ()
        args += [x.data_ptr(), *lead, *x.stride()[:-1], x.shape[-2], y.data_ptr(), *lead, *y.stride()[:-1]]
    x = q if q is not None else k
    B, S = (1, x.shape[0]) if x.dim() == 3 else x.shape[:2]
    p_sb, p_st = (0, pos.stride(0)) if pos.dim() == 1 else pos.stride()
    with _device(x, pos, freqs):
        _lib.check(_lib.load().dash_rope(
            *args, _TYPES[x.dtype], pos.data_ptr(), int(pos.dtype == torch.int64), p_sb, p_st,
            freqs.data_ptr(), freqs.numel(), start, int(interleaved), int(back), factor, B, S,
            x.shape[-1], _stream()), "dash_rope")
    return tuple(outs)


def apply_rope(q, k, positions, inv_freq, interleaved=False, start=0, factor=1.0):
    """q and k [T, heads, D] or [B, S, heads, D] (any strides; fp32, bf16 or fp16; k may be None) with
    the part [start, start + 2 len(inv_freq)) of every head row turned by its token's position times
    inv_freq, and scaled by factor; the rest as it is.  positions int32 or int64 [T], [S] or [B, S],
    whole numbers of up to 2^53 of either sign.  Returns new tensors (q', k'), or q' alone where k is
    None; differentiable in q and k, to any order, in forward mode too (torch.func's transforms are
    refused by torch).  D even, at most 256 pairs.  Under capture a leaf that an eager graph still
    refers to is refused (a captured backward pass of it would end the process)."""
    if q.dim() not in (3, 4):
        raise ValueError("q: [T, heads, D] or [B, S, heads, D] needed")
    lead = q.shape[:-2]
    if k is not None and (k.shape[:-2] != lead or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}")
    if positions.shape not in (lead, lead[-1:]):
        raise ValueError(f"positions {tuple(positions.shape)} of rows {tuple(lead)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions: int32 or int64")
    if q.dtype not in _TYPES or (k is not None and k.dtype != q.dtype):
        raise NotImplementedError("q and k of one type: fp32, bf16 or fp16")
    start = int(start)
    if inv_freq.dim() != 1:
        raise ValueError("inv_freq: [pairs] needed")
    _part(q.shape[-1], inv_freq.numel(), start)
    with _device(q, k, positions, inv_freq):
        freqs = _freqs(inv_freq)
    fresh = list(_leaves_in_capture(q, k)) if torch.is_grad_enabled() else ()
    q, k2 = _rope(q, k, positions, freqs, bool(interleaved), start, float(factor), False)
    del fresh
    return q if k is None else (q, k2)


def rope_append(q, k, v, positions, slots, k_cache, v_cache, inv_freq, interleaved=False, start=0,
                factor=1.0):
    """The new tokens of a step: q [T, H, D] turned as apply_rope does and returned; k [T, Hkv, D]
    turned and v as it is written to rows `slots` (int64 [T], kv_pages.step_rows; page * page_size +
    offset) of the caches [num_pages, page_size, Hkv, D], in place.  Tokens whose slot is none (-1)
    are not written.  Slots are distinct.  One type for all: fp32, bf16 or fp16; any strides with
    contiguous head rows.  For inference: no gradients."""
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[0] != q.shape[0] \
            or k.shape[2] != q.shape[2]:
        raise ValueError(f"q [T, H, D] and k, v [T, Hkv, D]: {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    T, H, D = q.shape
    Hkv = k.shape[1]
    _shape(positions, (T,), "positions")
    _shape(slots, (T,), "slots")
    if positions.dtype not in (torch.int32, torch.int64) or slots.dtype != torch.int64:
        raise ValueError("positions: int32 or int64, slots: int64")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or k_cache.shape[2:] != (Hkv, D) \
            or k_cache.shape[1] == 0:
        raise ValueError(f"caches [num_pages, page_size, {Hkv}, {D}]: {tuple(k_cache.shape)}, "
                         f"{tuple(v_cache.shape)}")
    if q.dtype not in _TYPES or any(x.dtype != q.dtype for x in (k, v, k_cache, v_cache)):
        raise NotImplementedError("q, k, v and the caches of one type: fp32, bf16 or fp16")
    if _derivatives(q, k, v, k_cache, v_cache):
        raise ValueError("rope_append writes a cache: no gradients (apply_rope has them)")
    for x in (k_cache, v_cache):
        if x.stride(3) != 1 and D > 1:
            raise ValueError("a cache with contiguous head rows is needed (written in place)")
        if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
            raise ValueError("a cache with overlapping rows (written in place)")
    start = int(start)
    if inv_freq.dim() != 1:
        raise ValueError("inv_freq: [pairs] needed")
    _part(D, inv_freq.numel(), start)
    with _device(q, k, v, positions, slots, k_cache, v_cache, inv_freq):
        freqs = _freqs(inv_freq)
        q, k, v = _inner(q), _inner(k), _inner(v)
        pos, at = positions.contiguous(), slots.contiguous()
        out = torch.empty(T, H, D, dtype=q.dtype, device=q.device)
        pages, page_size = k_cache.shape[:2]
        _lib.check(_lib.load().dash_rope_append(
            _ptr(q), *q.stride()[:2], H, _ptr(out), H * D, D, _ptr(k), *k.stride()[:2], _ptr(v),
            *v.stride()[:2], Hkv, _TYPES[q.dtype], _ptr(pos), int(pos.dtype == torch.int64),
            _ptr(at), _ptr(k_cache), *k_cache.stride()[:3], _ptr(v_cache), *v_cache.stride()[:3],
            page_size, pages, _ptr(freqs), freqs.numel(), start, int(interleaved), float(factor), T,
            D, _stream()), "dash_rope_append")
    return out
