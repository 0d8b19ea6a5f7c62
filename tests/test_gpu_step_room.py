"""Steps whose new tokens do not fit the batch (pipeline.start_step): refused as a whole.  Outputs against
64 bits as in test_gpu_answers.py, with its tolerance."""

import pytest
import torch

from ananta_ocr_amd import pipeline
from test_gpu_answers import DEV, I32, _close, _Serving

pytestmark = pytest.mark.gpu


def _state(s):
    return [x.clone() for x in (s.k, s.v, s.pool.table, s.pool.refs, s.pool.lens)]


@pytest.mark.parametrize("new, T", [([0, 5, 4], 8), ([9, 0, 0], 8), ([8, 1, 0], 8), ([1, 0, 0], 0),
                                    ([2 ** 31 - 1, 0, 0], 8), ([2 ** 31 - 1] * 3, 8), ([2 ** 31 - 9, 3, 6], 8)])
def test_more_tokens_than_rows(new, T):
    """Refused, nothing written, and the next step is the one that would have followed without it."""
    s = _Serving(16, 3, 60, 1, 21)
    first = [20, 33, 0]
    qkv = s.qkv(53)
    s.step(first, qkv, None, None, 53)
    s.reference(first, [0] * 3, qkv)
    before = _state(s)
    qkv = s.qkv(T)
    st, _ = s.step(new, qkv, None, None, T)
    assert st.ok.item() == 0 and st.slots.tolist() == [-1] * T
    assert all(torch.equal(a, b) for a, b in zip(before, _state(s)))
    assert st.context_lens.tolist() == first
    then = [2, 3, 3]
    qkv = s.qkv(8)
    st, outs = s.step(then, qkv, None, None, 8)
    assert st.ok.item() == 1 and s.pool.lens.tolist() == [22, 36, 3]
    _close(outs[0], s.reference(then, first, qkv)[0])


def test_as_many_tokens_as_rows():
    s = _Serving(16, 3, 60, 1, 22)
    qkv = s.qkv(12)
    st, outs = s.step([5, -4, 7], qkv, None, None, 12)
    assert st.ok.item() == 1 and s.pool.lens.tolist() == [5, 0, 7]
    assert bool((st.slots >= 0).all()) and st.seq.tolist() == [0] * 5 + [2] * 7
    _close(outs[0], s.reference([5, 0, 7], [0] * 3, qkv)[0])


def test_replays_with_and_without_room():
    """A captured step, replayed with lengths that fit and that do not, by turns."""
    s = _Serving(16, 4, 80, 1, 23)
    s.step([30, 0, 0, 0], s.qkv(30), None, None, 30)
    T = 6
    n = torch.zeros(4, dtype=I32, device=DEV)
    buf = s.qkv(T)

    def run():
        st = pipeline.start_step(s.pool, n, T)
        return st, [pipeline.shared_step(st, *x, s.k[l], s.v[l], s.pool.table, s.f) for l, x in enumerate(buf)]

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st, _ = run()
    lens = [30, 0, 0, 0]
    for new, fits in (([1, 2, 3, 0], True), ([3, 2, 1, 1], False), ([0, 0, 6, 0], True), ([7, 0, 0, 0], False),
                      ([2 ** 31 - 1, 2, 0, 0], False), ([1, 1, 1, 1], True)):
        n.copy_(torch.tensor(new, dtype=I32))
        before = _state(s)
        graph.replay()
        torch.cuda.synchronize()
        assert st.ok.item() == int(fits)
        if fits:
            lens = [a + b for a, b in zip(lens, new)]
        else:
            assert all(torch.equal(a, b) for a, b in zip(before, _state(s)))
        assert s.pool.lens.tolist() == lens


def test_many_rows():
    """The sum over all of the pool's rows, more than a work-group's threads."""
    s = _Serving(4, 3000, 3010, 1, 24)
    new = [1] * 3000
    st = pipeline.start_step(s.pool, torch.tensor(new, dtype=I32, device=DEV), 2999)
    assert st.ok.item() == 0 and not s.pool.lens.any()
    st = pipeline.start_step(s.pool, torch.tensor(new, dtype=I32, device=DEV), 3000)
    assert st.ok.item() == 1 and s.pool.lens.tolist() == new and bool((st.slots >= 0).all())
