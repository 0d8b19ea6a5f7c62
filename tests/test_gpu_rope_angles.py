"""Angles and factors of rotary positions (rope.apply_rope) against exact arithmetic.

A pair (1, 0) turns into (f cos a, f sin a), rounded once to the rows' 32 bits: off by half a step, 2^-24 of
its value.  The reference reduces position * frequency, a rational number, by a 2 pi of 70 digits, so that
its own cos and sin are off by 2^-52.  The kernel's are 64-bit series whose next terms are below 1.2e-10
(the cosine's; x^12 / 12! at pi / 4), of an angle of 64 bits, its turns off by a few 2^-53 whatever the
position (2 pi 4 2^-53 = 3e-15): f 1.3e-10 beside the half step."""

from fractions import Fraction
import math

import pytest
import torch

from ananta_ocr_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
TWO_PI = Fraction("6.283185307179586476925286766559005768394338798750211641949889184615633")


def _reference(pos, freqs):
    """(cos, sin) float64 [n, pairs] of whole positions."""
    turns = [[Fraction(p) * Fraction(f) / TWO_PI for f in freqs.tolist()] for p in pos.tolist()]
    part = torch.tensor([[float(t - round(t)) for t in row] for row in turns], dtype=torch.float64)
    # (a turn's part of 64 bits: its rounding of 2^-54 is 2^-51 of an angle)
    a = part * (2 * math.pi)
    return a.cos(), a.sin()


def _turned(pos, freqs, factor=1.0):
    m = freqs.numel()
    x = torch.zeros(len(pos), 1, 2 * m)
    x[..., :m] = 1.0
    y = rope.apply_rope(x.to(DEV), None, pos.to(DEV), freqs.to(DEV), factor=factor)[:, 0].double().cpu()
    return y[:, :m], y[:, m:]


def _check(pos, freqs, factor=1.0):
    for got, ref in zip(_turned(pos, freqs, factor), _reference(pos, freqs)):
        ref = ref * factor
        err = (got - ref).abs()
        tol = ref.abs() * 2.0 ** -24 + abs(factor) * 1.3e-10
        assert bool((err <= tol).all()), (err - tol).max().item()


@pytest.mark.parametrize("far", [0, 10 ** 5, 2 ** 31 - 300, -(2 ** 31), 2 ** 33, 2 ** 40, -(2 ** 47), 2 ** 53 - 300])
def test_far_positions(far):
    pos = far + torch.arange(300)
    _check(pos, torch.cat((torch.ones(1, dtype=torch.float64), rope.inv_freq(64)[0])))
    if abs(far) < 2 ** 31:
        _check(pos.to(torch.int32), rope.inv_freq(64)[0])


@pytest.mark.parametrize("factor", [1.3688879454113936, 1.0 / 3.0, -1.1, 1.0 + 2.0 ** -25])
def test_factors_of_64_bits(factor):
    """The first is that of a 40-fold stretch (0.1 ln 40 + 1).  Rounded to 32 bits it would be off by 3e-8 of
    itself, half a step more; the last would be 1."""
    _check(torch.arange(2000), rope.inv_freq(64)[0], factor)
    f = rope.inv_freq(64, device=DEV)[0]
    x = torch.ones(50, 1, 64, device=DEV)
    caches = torch.zeros(2, 1, 64, 1, 64, device=DEV)
    pos, slots = torch.arange(50, device=DEV), torch.arange(50, device=DEV)
    rope.rope_append(x, x, x, pos, slots, *caches, f, factor=factor)
    assert torch.equal(caches[0, 0, :50], rope.apply_rope(x, None, pos, f, factor=factor))
