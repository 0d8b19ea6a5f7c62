"""What rope.inv_freq takes of a configuration's rope_scaling.  No GPU calls."""

import math

import pytest
import torch

from ananta_ocr_amd import rope

YARN = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1}


def test_a_given_factor_of_the_attention():
    """It takes the place of the one that follows from the stretch, and of mscale's."""
    for more in ({}, {"mscale": 0.707, "mscale_all_dim": 0.5}):
        f, factor = rope.inv_freq(64, scaling={**YARN, **more, "attention_factor": 1.25})
        want, other = rope.inv_freq(64, scaling={**YARN, **more})
        assert factor == 1.25 and other != 1.25 and torch.equal(f, want)
    assert rope.inv_freq(64, scaling={**YARN, "attention_factor": None})[1] == 0.1 * math.log(40) + 1.0


def test_borders_of_the_ramp():
    """truncate false: the ramp runs between the indices themselves, not the whole numbers around them."""
    m, n, base = 32, 4096, 10000.0
    at = [m * math.log(n / (turns * 2 * math.pi)) / math.log(base) for turns in (32, 1)]
    for truncate in (True, False):
        f, _ = rope.inv_freq(2 * m, scaling={**YARN, "truncate": truncate})
        lo, hi = (math.floor(at[0]), math.ceil(at[1])) if truncate else at
        plain = [base ** (-j / m) for j in range(m)]
        ramp = [min(max((j - lo) / (hi - lo), 0.0), 1.0) for j in range(m)]
        want = torch.tensor([p / 40 * r + p * (1 - r) for p, r in zip(plain, ramp)], dtype=torch.float64)
        assert torch.allclose(f, want, rtol=1e-12)
    assert torch.equal(rope.inv_freq(2 * m, scaling=YARN)[0], rope.inv_freq(2 * m, scaling={**YARN, "truncate": True})[0])


def test_types_without_a_factor_of_the_attention():
    """They refuse one that is not 1."""
    for kind in ("linear", "ntk", "default"):
        assert rope.inv_freq(64, scaling={"rope_type": kind, "factor": 2, "attention_factor": 1.0})[1] == 1.0
        with pytest.raises(NotImplementedError):
            rope.inv_freq(64, scaling={"rope_type": kind, "factor": 2, "attention_factor": 1.25})
