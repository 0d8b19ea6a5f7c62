"""Tree steps over prefix sums and batches that do not fit the rows: the rows of the trees that are
there come out as without them, and nothing past the rows is touched."""

import math

import pytest
import torch

from ananta_ocr_amd import pipeline, tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
IDX = 128.0 / math.sqrt(128.0)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _step(width, seed=3, B=4, T=15):
    bs, H = 64, 2
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(8 * B, bs, H, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    ik = torch.randn(8 * B, bs, width, generator=g).to(DEV)
    hc = torch.randn(width, generator=g).to(DEV)
    table = torch.randperm(8 * B, generator=g).to(torch.int32).view(B, 8).to(DEV)
    ctx = _i32([7 * bs + 3, 6 * bs, 5 * bs + 1, 300][:B])
    state = pipeline.KBarPageCache(8 * B, width, DEV)
    state.put_sequences(ik, hc, bs, table, ctx)
    q = torch.randn(200, H, 128, generator=g).bfloat16().to(DEV)
    iq = torch.randn(200, width, generator=g).to(DEV)
    par = torch.randint(-3, 40, (200,), generator=g).to(torch.int32).to(DEV)

    def call(n, cu, most, rows=slice(None)):
        return pipeline.tree_step(state, q[:n], k, v, iq[:n], bs, 1, IDX, 1e-4, 1.0, 3, 4, table[rows],
                                  ctx[rows], _i32(cu), par[:n], most, out_dtype=torch.float32,
                                  return_routing=True)
    return call, state, iq, ctx, table


@pytest.mark.parametrize("width", [128, 64])
def test_prefix_sums_past_the_rows_are_cut(width):
    """The last trees claim rows there are not: the third is cut to the two there are, the fourth has
    none."""
    call = _step(width)[0]
    for most in (9, 200):
        want, (idx, bias, valid), pos = call(15, [0, 9, 13, 15, 15], most)
        for cu in ([0, 9, 13, 10 ** 6, 10 ** 6 + 5], [0, 9, 13, 16, 2 ** 31 - 1], [-7, 9, 13, 15, 14]):
            got, (idx2, bias2, valid2), pos2 = call(15, cu, most)
            assert torch.equal(got, want) and torch.equal(pos, pos2)
            assert torch.equal(valid, valid2) and torch.equal(bias, bias2)
            assert torch.equal(torch.where(valid, idx, -1), torch.where(valid2, idx2, -1))


def test_scores_write_their_rows_alone():
    """tree_scores of rows in the middle of a tensor that prefix sums reach past."""
    _, state, iq, ctx, table = _step(128)
    dep = torch.zeros(200, dtype=torch.int32, device=DEV)
    want = tree.tree_scores(iq[:140], _i32([0, 9, 13, 140, 140]), ctx, dep[:140], table, state.kbar, 64, 1, 127)
    got = tree.tree_scores(iq[:140], _i32([0, 9, 13, 10 ** 9, 5]), ctx, dep[:140], table, state.kbar, 64, 1, 250)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
