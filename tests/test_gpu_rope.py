"""Rotary positions (rope.apply_rope, rope.rope_append) against 64 bits.

Tolerance: with factor f, the pair (x, y) and u = 2^-24 the sine and cosine are off by u f (their
rounding) and u f (f's own), each product by u of itself and the sum by u of itself: at most 5 u f (|x| +
|y|) in all; 6 is stated.  Angles are products of 64 bits, reduced: off by at most 2^-51 of the angle, which
counts for far positions.  The result's type adds half a step of the value (fp16 also 2^-25, half its
smallest number)."""

import math

import pytest
import torch

from ananta_ocr_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _reference(x, pos, f, interleaved, start, factor, sign=1.0):
    """(turned rows in 64 bits, |x| + |y| of every element's pair, 0 where it is copied)."""
    m = f.numel()
    x = x.detach().double().cpu()
    pos = pos.cpu().expand(x.shape[:-2])
    a = (pos.double()[..., None] * f.cpu().double())[..., None, :] * sign
    c, s = a.cos() * factor, a.sin() * factor
    out, mag = x.clone(), torch.zeros_like(x)
    ix = torch.arange(m)
    i, j = (start + 2 * ix, start + 2 * ix + 1) if interleaved else (start + ix, start + m + ix)
    u, v = x[..., i], x[..., j]
    out[..., i], out[..., j] = u * c - v * s, v * c + u * s
    mag[..., i] = mag[..., j] = u.abs() + v.abs()
    return out, mag


def _close(y, x, pos, f, interleaved=False, start=0, factor=1.0, sign=1.0):
    ref, mag = _reference(x, pos, f, interleaved, start, factor, sign)
    far = float(pos.abs().max() if pos.numel() else 0) * float(f.max() if f.numel() else 0)
    tol = mag * abs(factor) * (6 * 2.0 ** -24 + far * 2.0 ** -51)
    if y.dtype != torch.float32:
        tol = tol * 1.01 + ref.abs() * torch.finfo(y.dtype).eps / 2
        tol = tol + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    err = (y.detach().double().cpu() - ref).abs()
    assert y.dtype == x.dtype and y.shape == x.shape
    assert bool((err <= tol).all()), (err - tol).max().item()
    still = mag == 0
    assert bool((y.detach().double().cpu()[still] == ref[still]).all())


CASES = [
    # tokens, H, Hkv, D, pairs, start
    (1, 1, 1, 128, 64, 0),
    (5, 10, 10, 128, 64, 0),
    (7, 10, 2, 128, 32, 64),
    (33, 3, 1, 128, 16, 32),
    (4, 2, 2, 64, 32, 0),
    (9, 2, 3, 48, 5, 6),              # a part that no 16 bytes fit
    (6, 5, 1, 34, 17, 0),
    (3, 1, 2, 2, 1, 0),
    (8, 2, 2, 512, 256, 0),           # the most pairs
    (300, 4, 4, 128, 0, 64),          # nothing to turn
    (0, 4, 4, 128, 64, 0),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype", TYPES)
def test_rope_against_64_bits(case, dtype, interleaved):
    T, H, Hkv, D, m, start = CASES[case]
    g = torch.Generator().manual_seed(case)
    q = torch.randn(T, H, D, generator=g).to(dtype).to(DEV)
    k = torch.randn(T, Hkv, D, generator=g).to(dtype).to(DEV)
    pos = torch.randint(-5, 10 ** 5, (T,), generator=g).to(DEV)
    f, _ = rope.inv_freq(2 * m, device=DEV)
    q2, k2 = rope.apply_rope(q, k, pos, f, interleaved=interleaved, start=start, factor=1.25)
    _close(q2, q, pos, f, interleaved, start, 1.25)
    _close(k2, k, pos, f, interleaved, start, 1.25)
    one = rope.apply_rope(q, None, pos.to(torch.int32), f, interleaved=interleaved, start=start, factor=1.25)
    assert torch.equal(one, q2)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_views(interleaved):
    """The pieces of one projection, heads before tokens, rows at odd addresses, broadcast positions."""
    g = torch.Generator().manual_seed(3)
    f, _ = rope.inv_freq(128, device=DEV)
    x = torch.randn(2, 9, 14, 128, generator=g).bfloat16().to(DEV)
    q, k, _ = x.split((10, 2, 2), 2)
    pos = torch.arange(4, 13, device=DEV)
    q2, k2 = rope.apply_rope(q, k, pos, f, interleaved)
    _close(q2, q, pos, f, interleaved)
    _close(k2, k, pos, f, interleaved)
    y = torch.randn(2, 3, 9, 128, generator=g).to(DEV).transpose(1, 2)       # heads first
    both = torch.stack((pos, pos * 7 + 2))
    y2 = rope.apply_rope(y, None, both, f, interleaved)
    _close(y2, y, both, f, interleaved)
    assert y2.stride() == y.stride()
    odd = torch.randn(2 * 9 * 3 * 131 + 1, generator=g).bfloat16().to(DEV)[1:].view(2, 9, 3, 131)[..., 1:129]
    _close(rope.apply_rope(odd, None, both, f, interleaved), odd, both, f, interleaved)
    apart = torch.randn(2, 9, 3, 256, generator=g).to(DEV)[..., ::2]         # elements apart
    _close(rope.apply_rope(apart, None, both, f, interleaved), apart, both, f, interleaved)
    same = torch.randn(2, 9, 1, 128, generator=g).to(DEV).expand(2, 9, 4, 128)
    _close(rope.apply_rope(same, None, both, f, interleaved), same, both, f, interleaved)


@pytest.mark.parametrize("far", [10 ** 6, 2 ** 31 - 1, -(2 ** 31), 2 ** 40])
def test_rope_far_positions(far):
    g = torch.Generator().manual_seed(5)
    f, _ = rope.inv_freq(64, device=DEV)
    x = torch.randn(6, 2, 64, generator=g).to(DEV)
    pos = far + torch.tensor([0, -1, -2, -1000, -54321, -99999], device=DEV)
    if far == -(2 ** 31):
        pos = pos + 99999
    _close(rope.apply_rope(x, None, pos, f), x, pos, f)
    if abs(far) < 2 ** 32:
        _close(rope.apply_rope(x, None, pos.to(torch.int32), f), x, pos, f)


def test_rope_values_that_are_not_finite():
    """A row that is not finite leaves the others, and what is only copied, alone."""
    f, _ = rope.inv_freq(64, device=DEV)
    x = torch.ones(3, 2, 128, device=DEV).bfloat16()
    x[1, 0, 5] = math.nan
    x[2, 1, 100] = math.inf
    y = rope.apply_rope(x, None, torch.arange(3, device=DEV), f)
    assert torch.isnan(y).sum() == 2 and y[2, 1, 100] == math.inf
    assert bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2, 0]).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rope_gradients(dtype, interleaved):
    """Against the formula's, in one and both inputs, from broadcast gradients, and the second order."""
    g = torch.Generator().manual_seed(7)
    f, _ = rope.inv_freq(32, device=DEV)
    q = torch.randn(2, 5, 3, 64, generator=g).to(dtype).to(DEV).requires_grad_()
    k = torch.randn(2, 5, 1, 64, generator=g).to(dtype).to(DEV).requires_grad_()
    pos = torch.randint(0, 5000, (2, 5), generator=g).to(DEV)
    how = dict(interleaved=interleaved, start=16, factor=1.5)
    dq = torch.randn(2, 5, 3, 64, generator=g).to(dtype).to(DEV)
    dk = torch.randn(2, 5, 1, 64, generator=g).to(dtype).to(DEV)
    q2, k2 = rope.apply_rope(q, k, pos, f, **how)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk), retain_graph=True)
    _close(gq, dq, pos, f, sign=-1.0, **how)
    _close(gk, dk, pos, f, sign=-1.0, **how)
    only, = torch.autograd.grad(k2, (k,), (dk,), retain_graph=True)
    assert torch.equal(only, gk)
    gq, gk = torch.autograd.grad(q2.sum(), (q, k), allow_unused=True)
    assert gk is None
    _close(gq, torch.ones_like(q), pos, f, sign=-1.0, **how)
    # a shared head: the gradient of its copies is their sum
    one = torch.randn(2, 5, 1, 64, generator=g).to(DEV).requires_grad_()
    y = rope.apply_rope(one.expand(2, 5, 4, 64), None, pos, f, **how)
    up = torch.randn(2, 5, 4, 64, generator=g).to(DEV)
    got, = torch.autograd.grad(y, one, up)
    want, mag = _reference(up, pos, f, interleaved, 16, 1.5, -1.0)
    # (each of the four as above, and the sum of four in 32 bits)
    tol = (1.5 * 6 * mag + 4 * want.abs()).sum(2, keepdim=True) * 2.0 ** -24
    assert bool(((got.double().cpu() - want.sum(2, keepdim=True)).abs() <= tol).all())
    # the gradient's gradient turns forward again
    w = torch.randn(2, 5, 3, 64, generator=g).to(dtype).to(DEV).requires_grad_()
    q2 = rope.apply_rope(q, None, pos, f, **how)
    gq, = torch.autograd.grad(q2, q, w, create_graph=True)
    back, = torch.autograd.grad(gq, w, dq)
    _close(back, dq, pos, f, **how)


def test_rope_gradient_against_differences():
    g = torch.Generator().manual_seed(8)
    f, _ = rope.inv_freq(8, device=DEV)
    x = torch.randn(3, 2, 10, generator=g).to(DEV)
    up = torch.randn(3, 2, 10, generator=g).to(DEV)
    pos = torch.tensor([0, 3, 77], device=DEV)
    y = x.clone().requires_grad_()
    got, = torch.autograd.grad(rope.apply_rope(y, None, pos, f, start=2), y, up)
    # the map is linear: differences of any step are exact but for roundings of 2^-24 of ~60 sums
    for i in range(x.numel()):
        e = torch.zeros_like(x).view(-1)
        e[i] = 1.0
        d = rope.apply_rope(x + e.view_as(x), None, pos, f, start=2) - rope.apply_rope(x, None, pos, f, start=2)
        assert abs(float((d.double() * up.double()).sum()) - float(got.view(-1)[i])) < 60 * 6 * 2.0 ** -23


def test_rope_backward_in_a_graph():
    """Forward and backward captured, once the eager graph of the same leaf is gone (while it lives the
    call is refused: test_rope_host.py); replays against eager."""
    f, _ = rope.inv_freq(64, device=DEV)
    x = torch.randn(12, 2, 64, device=DEV).requires_grad_()
    up = torch.randn(12, 2, 64, device=DEV)
    pos = torch.arange(12, device=DEV)
    eager = rope.apply_rope(x, None, pos, f)
    del eager
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        torch.autograd.grad(rope.apply_rope(x, None, pos, f), x, up)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = rope.apply_rope(x, None, pos, f)
        dx, = torch.autograd.grad(y, x, up)
    for seed in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(12, 2, 64, generator=torch.Generator().manual_seed(seed)))
            up.copy_(torch.randn(12, 2, 64, generator=torch.Generator().manual_seed(seed + 9)))
            pos.add_(13)
        graph.replay()
        torch.cuda.synchronize()
        _close(y, x, pos, f)
        _close(dx, up, pos, f, sign=-1.0)
        x2 = x.detach().clone().requires_grad_()
        g2, = torch.autograd.grad(rope.apply_rope(x2, None, pos, f), x2, up)
        assert torch.equal(g2, dx)


APPEND = [
    # T, H, Hkv, D, pairs, start, page, pages
    (1, 2, 2, 128, 64, 0, 64, 3),
    (8, 10, 10, 128, 64, 0, 64, 5),
    (37, 10, 2, 128, 32, 64, 16, 7),
    (70, 3, 1, 64, 16, 0, 1, 90),
    (9, 2, 2, 20, 5, 4, 7, 4),
    (0, 2, 2, 128, 64, 0, 64, 3),
    (5, 2, 2, 128, 64, 0, 64, 0),     # a pool without pages: nothing is written
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case, dtype, interleaved):
    """Rows in their slots, everything else of the caches as it was, tokens without a slot left out."""
    T, H, Hkv, D, m, start, page, pages = APPEND[case]
    g = torch.Generator().manual_seed(case + 50)
    x = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV)
    q, k, v = x.split((H, Hkv, Hkv), 1)
    # a layer of a cache whose token rows hold more than this pool's heads
    wide = torch.randn(2, pages, page, 2, Hkv, D, generator=g).to(dtype).to(DEV)
    kc, vc = wide[1, :, :, 0], wide[1, :, :, 1]
    before = wide.clone()
    pos = torch.randint(0, 30000, (T,), generator=g).to(DEV)
    slots = torch.randperm(max(pages * page, T), generator=g)[:T]
    if T > 2:
        slots[1], slots[2] = -1, pages * page + 5
    slots = slots.to(DEV)
    f, _ = rope.inv_freq(2 * m, device=DEV)
    out = rope.rope_append(q, k, v, pos, slots, kc, vc, f, interleaved=interleaved, start=start)
    _close(out, q, pos, f, interleaved, start)
    k2 = rope.apply_rope(k, None, pos, f, interleaved=interleaved, start=start)
    _close(k2, k, pos, f, interleaved, start)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            before[1, s // page, s % page, 0] = k2[t]
            before[1, s // page, s % page, 1] = v[t]
    assert torch.equal(wide, before)


def test_append_in_a_graph_and_on_streams():
    """Captured, replayed with other positions and slots between eager calls, and on another stream."""
    g = torch.Generator().manual_seed(11)
    f, _ = rope.inv_freq(128, device=DEV)
    x = torch.randn(8, 6, 128, generator=g).bfloat16().to(DEV)
    q, k, v = x.split((2, 2, 2), 1)
    kc, vc = (torch.zeros(4, 16, 2, 128, device=DEV).bfloat16() for _ in range(2))
    pos, slots = torch.arange(8, device=DEV, dtype=torch.int32), torch.arange(8, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rope.rope_append(q, k, v, pos, slots, kc, vc, f)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.rope_append(q, k, v, pos, slots, kc, vc, f)
    for i in range(3):
        pos.add_(5)
        slots.add_(17)
        k2, v2 = kc.clone(), vc.clone()
        want = rope.rope_append(q, k, v, pos, slots, k2, v2, f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kc, k2) and torch.equal(vc, v2)
