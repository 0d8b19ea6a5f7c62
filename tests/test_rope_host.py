"""Rotary frequencies, and what the rotary calls refuse.  No GPU calls."""

import math

import pytest
import torch

from ananta_ocr_amd import rope


def test_frequencies():
    f, factor = rope.inv_freq(64, 10000.0)
    assert factor == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([10000.0 ** (-j / 32) for j in range(32)], dtype=torch.float64))
    half, _ = rope.inv_freq(64, scaling={"type": "linear", "factor": 4})
    assert torch.allclose(half, f / 4)
    ntk, _ = rope.inv_freq(64, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    assert rope.inv_freq(0)[0].numel() == 0


@pytest.mark.parametrize("s", [1, 8, 40])
def test_frequencies_of_yarn(s):
    """Frequencies of many turns over the original length stay, those of few are divided."""
    n, dim = 4096, 64
    f, _ = rope.inv_freq(dim)
    y, factor = rope.inv_freq(dim, scaling={"type": "yarn", "factor": s, "original_max_position_embeddings": n,
                                            "beta_fast": 32, "beta_slow": 1, "mscale": 1.0, "mscale_all_dim": 0})
    turns = f * n / (2 * math.pi)
    ratio = y / f
    assert torch.allclose(ratio[turns > 40], torch.ones(1, dtype=torch.float64))
    assert torch.allclose(ratio[turns < 0.6], torch.full((1,), 1.0 / s, dtype=torch.float64))
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all())
    assert math.isclose(factor, 0.1 * math.log(s) + 1.0 if s > 1 else 1.0)
    same = rope.inv_freq(dim, scaling={"type": "yarn", "factor": s, "original_max_position_embeddings": n,
                                       "mscale": 0.7, "mscale_all_dim": 0.7})
    assert same[1] == 1.0


def test_refusals():
    q, k, pos = torch.zeros(4, 2, 16), torch.zeros(4, 1, 16), torch.arange(4)
    f, _ = rope.inv_freq(16)
    slots = torch.arange(4)
    kc = torch.zeros(2, 4, 1, 16)
    ok = dict(q=q, k=k, positions=pos, inv_freq=f)
    for bad, err in ((dict(q=q[0]), ValueError), (dict(k=k[:3]), ValueError), (dict(k=k[..., :8]), ValueError),
                     (dict(positions=pos[:3]), ValueError), (dict(positions=pos.float()), ValueError),
                     (dict(k=k.double()), NotImplementedError), (dict(q=q.double()), NotImplementedError),
                     (dict(start=1), ValueError), (dict(start=-1), ValueError),
                     (dict(inv_freq=f[None]), ValueError),
                     (dict(q=torch.zeros(4, 2, 17), k=None), NotImplementedError),
                     (dict(q=torch.zeros(4, 2, 600), k=None, inv_freq=rope.inv_freq(514)[0]), NotImplementedError),
                     (dict(), ValueError)):                  # (last: tensors of the CPU)
        with pytest.raises(err):
            rope.apply_rope(**{**ok, **bad})
    ok = dict(q=q, k=k, v=k, positions=pos, slots=slots, k_cache=kc, v_cache=kc.clone(), inv_freq=f)
    for bad, err in ((dict(v=k[:, :, :8]), ValueError), (dict(slots=slots.int()), ValueError),
                     (dict(slots=slots[:2]), ValueError), (dict(k_cache=kc[..., :8]), ValueError),
                     (dict(k_cache=kc[:1]), ValueError), (dict(v=k.bfloat16()), NotImplementedError),
                     (dict(k_cache=kc.bfloat16()), NotImplementedError),
                     (dict(k_cache=kc[:, :1].expand(2, 4, 1, 16)), ValueError),
                     (dict(k_cache=torch.zeros(2, 4, 1, 32)[..., ::2]), ValueError),
                     (dict(q=q.clone().requires_grad_()), ValueError), (dict(), ValueError)):
        with pytest.raises(err):
            rope.rope_append(**{**ok, **bad})
    for scaling in ({"type": "linear", "factor": 0}, {"type": "linear", "factor": -2}):
        with pytest.raises(ValueError):
            rope.inv_freq(16, scaling=scaling)
    with pytest.raises(NotImplementedError):
        rope.inv_freq(16, scaling={"type": "other"})
    with pytest.raises(ValueError):
        rope.inv_freq(15)


def test_leaves_under_capture(monkeypatch):
    """A leaf whose eager graph is alive is refused; one without is taken, also twice in a capture."""
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    monkeypatch.setattr(rope, "_stream", lambda: 5)
    x = torch.zeros(3, requires_grad=True)
    y = x * 2
    with pytest.raises(RuntimeError, match="eager graph"):
        list(rope._leaves_in_capture(x, None))
    del y
    fresh = list(rope._leaves_in_capture(None, x))
    assert len(fresh) == 1
    y = x * 2                                                # the captured graph refers to it
    del fresh
    assert list(rope._leaves_in_capture(x)) == []
    monkeypatch.setattr(rope, "_stream", lambda: 6)          # another capture, on another stream
    with pytest.raises(RuntimeError, match="eager graph"):
        list(rope._leaves_in_capture(x))
    del y
    assert list(rope._leaves_in_capture(x * 1, torch.zeros(2))) == []
