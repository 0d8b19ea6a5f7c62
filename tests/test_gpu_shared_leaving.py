"""The prompt of a group whose first answers have left (shared_prefix.attn_shared): it is read through a
sequence that takes part and holds it.  Against 64 bits, with the tolerances of test_gpu_shared.py and
test_gpu_answers.py."""

import pytest
import torch

from test_gpu_answers import DEV, I32, _close, _Serving
from test_gpu_shared import _case, _check, _padded, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [7, 80])
@pytest.mark.parametrize("reused", [False, True])
def test_the_first_answer_leaves(rows, reused):
    """A prompt of three answers: the first is freed, and in turn its row becomes another prompt's, while the
    group's prefix sums stay."""
    page = 16
    s = _Serving(page, rows, 250, 1, 31)
    rest = [0] * (rows - 5)
    new = [83, 60, 0, 0, 0] + rest
    qkv = s.qkv(sum(new))
    s.step(new, qkv, None, None, sum(new))
    s.reference(new, [0] * rows, qkv)
    i = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    assert s.pool.fork(i([0, 0, 0]), i([2, 3, 4])).item() == 1
    for b in (2, 3, 4):
        s.keys[0][b] = list(s.keys[0][0])
    groups, prefix = i([2, 5]), i([80])
    lens = [83, 60, 83, 83, 83] + rest

    def step(new):
        qkv = s.qkv(sum(new))
        st, outs = s.step(new, qkv, groups, prefix, sum(new))
        assert st.ok.item() == 1
        _close(outs[0], s.reference(new, lens, qkv)[0])
        for b, n in enumerate(new):
            lens[b] += n

    step([0, 0, 1, 1, 2] + rest)
    keep = s.pool.lens.clone()
    keep[2] = lens[2] = 0
    s.pool.free(keep)
    s.keys[0][2] = []
    step([0, 0, 0, 2, 1] + rest)
    if reused:
        assert s.pool.fork(i([1]), i([2])).item() == 1
        lens[2] = 60
    step([0, 0, 0, 1, 1] + rest)
    keep = s.pool.lens.clone()                       # the second one leaves as well
    keep[3] = lens[3] = 0
    s.pool.free(keep)
    s.keys[0][3] = []
    step([0, 0, 0, 0, 3] + rest)


@pytest.mark.parametrize("many", [0, 70])
@pytest.mark.parametrize("entry", [-1, 10 ** 8, 0])
def test_first_sequences_that_do_not_hold_the_prompt(entry, many):
    """Without rows and with a table row of nothing, or with rows that end before the prompt does."""
    c = _case([(500, [(600, 0), (20, 3), (600, 1), (499, 2), (700, 1)]), (128, [(128, 0), (130, 1)])], 4, 2, 64, 32)
    c["table"][0] = entry
    c["ctx"][0] = 0
    c["table"][1, 1:] = entry                        # (23 keys: one page)
    c["table"][5] = entry
    c = _padded(c, many) if many else c
    _check(c, *_run(c, return_lse=True))


def test_a_prompt_that_only_shorter_sequences_hold():
    """A prefix past every context: read through the longest, as far as any row sees."""
    c = _case([(400, [(400, 0), (90, 2), (300, 3), (200, 1)])], 2, 2, 64, 33)
    c["table"][0] = -1
    c["table"][1, 2:] = -1
    c["table"][3, 4:] = -1
    _check(c, *_run(c, return_lse=True))
