"""Sampling on the HIP kernels (csrc/dash_sample.hip): the next token of every row of logits from given
random numbers, and the probabilities that temperature, top-k, top-p and min-p leave, which are what
tree.verify_tree takes of a target and of a draft.

Token v of a row has the weight exp((x_v - M) / temperature), M the row's largest logit.  In the order of
falling logits, of equals the lower id first,

* the first top_k tokens stay (0 or below: all);
* of those the ones whose predecessors hold less than top_p of the weight of the first top_k (1 or
  above: all);
* of those the ones whose weight is at least min_p, which is min_p times the best token's (0 or below: all).

The first always does.  A temperature that is not above 0 keeps the first alone.  Logits of -inf and NaN
are masked; +inf counts as the largest number of 32 bits.  Weights are whole numbers of 2^-s of the best token's, s =
62 - ceil(log2 V) but at most 51, so that sums are exact and no result depends on how a launch ran; a token
below half of that counts as none (of 131,072, one more than 31.9 temperatures below the best).

Uniforms, temperature, top_p and min_p are taken in 32 bits, as are logits of other types than fp32, bf16 and fp16:
what has 64 is rounded.  (A uniform that so becomes 1 draws the last token that stays.)
"""

import ctypes
import functools

import torch

from . import _lib
from .ops import _ptr, _stream
from .tree import _derivatives, _device, _shape

MAX_VOCABULARY = 2 ** 20
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@functools.lru_cache(maxsize=256)
def _workspace(R, V):
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().dash_sample_workspace_size(R, V, nbytes), "workspace")
    return nbytes.value


def _floats(x, R, what):
    """(tensor or None, number)."""
    if not torch.is_tensor(x):
        return None, float(x)
    _shape(x, (R,), what)
    return x, 0.0


def _sample(logits, uniforms, temperature, top_k, top_p, min_p, probs_dtype):
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits: [R, V] needed")
    R, V = logits.shape
    if V > MAX_VOCABULARY:
        raise NotImplementedError(f"vocabularies of at most {MAX_VOCABULARY} tokens, got {V}")
    if probs_dtype is not None and probs_dtype not in _TYPES:
        raise NotImplementedError("probabilities in fp32, bf16 or fp16")
    if probs_dtype is not None and _derivatives(logits):
        raise ValueError("the probabilities have no gradients (detach the logits)")
    if uniforms is not None:
        _shape(uniforms, (R,), "uniforms")
    t, t0 = _floats(temperature, R, "temperature")
    p, p0 = _floats(top_p, R, "top_p")
    m, m0 = _floats(min_p, R, "min_p")
    k, k0 = None, 0
    if torch.is_tensor(top_k):
        _shape(top_k, (R,), "top_k")
        if top_k.is_floating_point() or top_k.dtype == torch.bool:
            raise ValueError("top_k: whole numbers")
        k = top_k
    else:
        k0 = max(0, min(int(top_k), 2 ** 31 - 1))
    with _device(logits, uniforms, t, k, p, m):
        x = logits if logits.dtype in _TYPES else logits.float()
        if x.stride(1) != 1 and V > 1:
            x = x.contiguous()
        u, t, p, m = (None if y is None else y.float().contiguous() for y in (uniforms, t, p, m))
        if k is not None:
            if k.dtype != torch.int32:           # (widened first: the bound fits no narrower type)
                k = k.to(torch.int64).clamp(0, 2 ** 31 - 1).to(torch.int32)
            k = k.contiguous()
        token = None if u is None else torch.empty(R, dtype=torch.int64, device=x.device)
        probs = None if probs_dtype is None else torch.empty(R, V, dtype=probs_dtype, device=x.device)
        if R:
            nbytes = _workspace(R, V)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            _lib.check(_lib.load().dash_sample(
                x.data_ptr(), x.stride(0), _TYPES[x.dtype], _ptr(u), _ptr(t), t0, _ptr(k), k0, _ptr(p), p0,
                _ptr(m), m0, R, V, _ptr(token), _ptr(probs), V, _TYPES.get(probs_dtype, 0), ws.data_ptr(),
                nbytes, _stream()), "dash_sample")
    return token, probs


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_probs=False,
           probs_dtype=torch.float32):
    """The next token of every row of logits [R, V] (fp32, bf16 or fp16): int64 [R].  The row's uniform
    (uniforms [R], in [0, 1)) draws among the tokens that stay: the first id whose running sum of weights
    exceeds it times the whole.  A uniform that is not above 0 counts as 0, one of 1 or more draws the last
    token that stays.  temperature, top_k, top_p and min_p are numbers or [R] tensors, a value for every
    row.  A row without any token (all masked) gives -1.  With return_probs also the probabilities [R, V]
    that are left (probs_dtype; a row without any token: zeros).  V at most 2^20."""
    if uniforms is None:
        raise ValueError("uniforms [R] are needed (token_probs does without)")
    token, probs = _sample(logits, uniforms, temperature, top_k, top_p, min_p,
                           probs_dtype if return_probs else None)
    return (token, probs) if return_probs else token


def token_probs(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dtype=torch.float32):
    """The probabilities [R, V] of the tokens after temperature, top-k, top-p and min-p (as sample draws
    from them), 0 for those that do not stay: the target, or the draft, of tree.verify_tree.  No gradients."""
    return _sample(logits, None, temperature, top_k, top_p, min_p, dtype)[1]
