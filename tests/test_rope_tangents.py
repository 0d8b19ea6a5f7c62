"""Forward-mode derivatives of rope.apply_rope.  On the CPU with the launch replaced by the formula in torch, which shows
where tangents go; on the GPU against the turn of the tangent, which is the map's derivative (it is linear)."""

import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from ananta_ocr_amd import rope


def _plain(q, k, pos, freqs, interleaved, start, factor, back):
    """rope._turn of rows [T, heads, 2 m], halves, without a graph and without tangents, as a launch is."""
    outs = []
    for x in (q, k):
        if x is None:
            outs.append(None)
            continue
        with torch.no_grad():
            x = forward_ad.unpack_dual(x).primal.detach()
            a = (pos.double()[:, None, None] * freqs * (-1 if back else 1))
            c, s, m = a.cos() * factor, a.sin() * factor, freqs.numel()
            u, v = x[..., :m], x[..., m:]
            outs.append(torch.cat((u * c - v * s, v * c + u * s), -1).to(x.dtype))
    return tuple(outs)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(rope, "_turn", _plain)
        monkeypatch.setattr(rope, "_device", lambda *a: contextlib.nullcontext())
        monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    return request.param


def _case(dev):
    g = torch.Generator().manual_seed(2)
    f, _ = rope.inv_freq(16, device=dev)
    rows = [torch.randn(5, n, 16, generator=g).to(dev) for n in (3, 2, 3, 2)]
    return *rows, torch.arange(5, device=dev) * 7, f


def _tangent(x):
    return forward_ad.unpack_dual(x).tangent


@pytest.mark.parametrize("grad", [False, True])
def test_tangents(dev, grad):
    """Of q, k and both, also where gradients are recorded."""
    q, k, tq, tk, pos, f = _case(dev)
    want_q, want_k = rope.apply_rope(tq, tk, pos, f, factor=1.25)
    if grad:
        q.requires_grad_(), k.requires_grad_()
    with forward_ad.dual_level():
        y = rope.apply_rope(forward_ad.make_dual(q, tq), None, pos, f, factor=1.25)
        assert torch.equal(_tangent(y), want_q)
        yq, yk = rope.apply_rope(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), pos, f, factor=1.25)
        assert torch.equal(_tangent(yq), want_q) and torch.equal(_tangent(yk), want_k)
        yq, yk = rope.apply_rope(q, forward_ad.make_dual(k, tk), pos, f, factor=1.25)
        assert torch.equal(_tangent(yk), want_k)
        assert _tangent(yq) is None or not _tangent(yq).any()
        yq, yk = rope.apply_rope(forward_ad.make_dual(q, tq), k, pos, f, factor=1.25)
        assert torch.equal(_tangent(yq), want_q)
        assert _tangent(yk) is None or not _tangent(yk).any()
        plain = rope.apply_rope(q, None, pos, f, factor=1.25)
        assert _tangent(plain) is None
        primal = forward_ad.unpack_dual(y).primal
    assert torch.equal(primal, plain)


def test_tangents_of_gradients(dev):
    """Forward over reverse: the gradient of (y w).sum() is w turned back, its tangent that of w's."""
    q, _, w, _, pos, f = _case(dev)
    tw = torch.randn(5, 3, 16, generator=torch.Generator().manual_seed(3)).to(dev)
    x = q.clone().requires_grad_()
    with forward_ad.dual_level():
        got, = torch.autograd.grad(rope.apply_rope(x, None, pos, f), x, forward_ad.make_dual(w, tw))
        tangent = _tangent(got)
        assert tangent is not None
    for u, v in ((w, got), (tw, tangent)):
        y = torch.zeros_like(q).requires_grad_()
        want, = torch.autograd.grad(rope.apply_rope(y, None, pos, f), y, u)
        assert torch.equal(v.detach(), want)


def test_gradients_of_tangents(dev):
    """Reverse over forward: the tangent of the output, as a function of the tangent given."""
    q, _, tq, up, pos, f = _case(dev)
    up = torch.randn(5, 3, 16, generator=torch.Generator().manual_seed(4)).to(dev)
    tq.requires_grad_()
    with forward_ad.dual_level():
        y = rope.apply_rope(forward_ad.make_dual(q, tq), None, pos, f)
        got, = torch.autograd.grad(_tangent(y), tq, up)
    z = q.clone().requires_grad_()
    want, = torch.autograd.grad(rope.apply_rope(z, None, pos, f), z, up)
    assert torch.equal(got, want)
