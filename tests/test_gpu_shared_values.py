"""Values that are not finite in partial sums of small weight (shared_prefix.attn_shared): a key that a row
sees reaches its output, whatever the other keys' scores are and wherever the work was cut.

Scores: the query is 40 in element 0 alone, a key -40 or 0 there, so that a score is -1600 / 11.3 = -141 or
0.  exp(-141) is 2^-204, which 32 bits do not hold: the partial sums of such keys alone have weight 0 beside
the others'.  Where every key that a row sees has the same score the output is the mean of their values."""

import math

import pytest
import torch

from test_gpu_shared import _case, _run

pytestmark = pytest.mark.gpu


def _far(groups, H, Hkv, page, low, alone=()):
    """_case with keys whose score is -141 where low(sequence, key), and 0 elsewhere."""
    c = _case(groups, H, Hkv, page, 40, alone=alone)
    c["q"].zero_()
    c["q"][..., 0] = 40.0
    for b, (k, _) in enumerate(c["keys"]):
        k.zero_()
        for j in range(len(k)):
            k[j, :, 0] = -40.0 if low(b, j) else 0.0
            c["k"][int(c["table"][b, j // page]), j % page] = k[j]
    return c


def _slot(c, b, j, page):
    return int(c["table"][b, j // page]), j % page


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("shared", [True, False])
def test_a_seen_value_of_weight_0(value, shared):
    """In the prompt, all of whose keys lie far below the sequences' own: every row sees it.  The prompt's
    sums are partials of their own, with and without a group."""
    c = _far([(640, [(700, 2), (650, 3)])], 4, 2, 64, lambda b, j: j < 640)
    clean = _run(c, groups=shared)
    assert bool(torch.isfinite(clean).all())
    c["v"][_slot(c, 0, 100, 64)][1, 7] = value
    if not shared:
        c["v"][_slot(c, 1, 100, 64)][1, 7] = value
    out = _run(c, groups=shared)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, 2:, 7] = True                             # the two query heads of key head 1
    assert torch.equal(~torch.isfinite(out), bad)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("more", [0, 3, 40, 90])
def test_whatever_else_is_in_the_batch(more):
    """A sequence of 2,000 keys, the first 1,900 far below the others, alone and beside other sequences (the
    work is cut elsewhere)."""
    c = _far([], 2, 2, 64, lambda b, j: b == 0 and j < 1900, alone=((2000, 1),) + ((300, 1),) * more)
    c["v"][_slot(c, 0, 1000, 64)][0, 3] = math.inf
    out = _run(c, groups=False)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 0, 3] = True
    assert torch.equal(~torch.isfinite(out), bad)


def test_an_unseen_value_stays_out():
    """Rows before the key: of their own sequence, in a partial of another run, and in other sequences."""
    c = _far([(128, [(1000, 5), (130, 2)])], 2, 1, 64, lambda b, j: j < 900)
    clean = _run(c)
    c["v"][_slot(c, 0, 1003, 64)][0, 9] = math.nan   # of row 3
    out = _run(c)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[3:5, :, 9] = True
    assert torch.equal(~torch.isfinite(out), bad) and torch.equal(out[~bad], clean[~bad])
