"""Slots of a step's new tokens (kv_pages.step_rows) against lists."""

import random

import pytest
import torch

from ananta_ocr_amd import kv_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _lists(table, ctx, new, page, pages, rows, lens=None):
    cu, seq, pos, slot = [0], [], [], []
    for b, n in enumerate(new):
        for t in range(ctx[b], ctx[b] + max(n, 0)):
            if len(seq) == rows:
                break
            ok = 0 <= t < 2 ** 31
            p = table[b][t // page] if ok and t // page < len(table[b]) else -1
            in_row = lens is None or t < lens[b]
            seq.append(b)
            pos.append(t if ok else -1)
            slot.append(p * page + t % page if 0 <= p < pages and in_row else -1)
        cu.append(len(seq))
    pad = [-1] * (rows - len(seq))
    return cu, seq + pad, pos + pad, slot + pad


def _check(table, ctx, new, page, pages, rows, lens=None):
    t = torch.tensor(table, dtype=torch.int32).view(len(ctx), -1)
    i32 = dict(dtype=torch.int32, device=DEV)
    got = kv_pages.step_rows(t.to(DEV), torch.tensor(ctx, **i32), torch.tensor(new, **i32), page, pages, rows,
                             None if lens is None else torch.tensor(lens, **i32))
    for x, y in zip(got, _lists(table, ctx, new, page, pages, rows, lens)):
        assert x.tolist() == y
    assert [x.dtype for x in got] == [torch.int32] * 3 + [torch.int64]


@pytest.mark.parametrize("B,n_hi,page,spare", [(1, 1, 64, 0), (8, 1, 64, 8), (5, 40, 7, 3), (300, 3, 16, 1),
                                               (64, 0, 64, 5), (1000, 2, 1, 0), (17, 300, 64, 255),
                                               (8192, 1, 64, 0)])
def test_against_lists(B, n_hi, page, spare):
    rng = random.Random(B * 31 + n_hi)
    ctx = [rng.randrange(0, 900) for _ in range(B)]
    new = [rng.randint(0, n_hi) for _ in range(B)]
    P = (900 + n_hi + page - 1) // page
    pages = 4 * B
    table = [[rng.randrange(-1, pages) for _ in range(P)] for _ in range(B)]
    _check(table, ctx, new, page, pages, sum(new) + spare)


def test_edges():
    table = [[3, 1], [2, 9], [0, -1], [4, 5]]
    _check(table, [5, 0, 6, -2], [3, 20, 4, 5], 8, 6, 40)            # past the table, no pages, before the start
    _check(table, [5, 0, 6, 0], [3, 5, -4, 2], 8, 6, 6)              # more than the rows; below 0: none
    _check(table, [0, 0, 0, 0], [0, 0, 0, 0], 8, 6, 0)
    _check(table, [0, 0, 0, 0], [2 ** 31 - 1] * 4, 8, 6, 5)          # sums past 32 bits
    _check(table, [2 ** 31 - 2, 1, 2, 3], [4, 1, 1, 1], 8, 6, 9)     # positions past 32 bits
    _check(table, [5, 0, 6, 1], [3, 2, 2, 2], 8, 6, 12, lens=[7, 2, 0, 9])
    got = kv_pages.step_rows(torch.zeros(0, 3, dtype=torch.int32, device=DEV), *(2 * [torch.zeros(
        0, dtype=torch.int32, device=DEV)]), 8, 6, 4)
    assert [x.tolist() for x in got] == [[0], [-1] * 4, [-1] * 4, [-1] * 4]
    _check([[], []], [0, 3], [1, 1], 8, 6, 3)


def test_slots_of_a_large_pool():
    """Slots past 32 bits."""
    table = torch.tensor([[2 ** 30, 7]], dtype=torch.int32, device=DEV)
    one = torch.tensor([3], dtype=torch.int32, device=DEV)
    assert kv_pages.step_rows(table, one, one, 64, 2 ** 30 + 1, 3)[3].tolist() == [2 ** 36 + 3, 2 ** 36 + 4,
                                                                                  2 ** 36 + 5]


def test_pool_rows_after_a_refused_reserve():
    """Rows share a last page until their growth gets pages of its own: where that was refused their new
    tokens have no slot, even though the shared page has room."""
    caches = kv_pages.PageCaches([torch.zeros(4, 8, 4, device=DEV)])
    pool = kv_pages.PagePool(caches, 3, 4)
    lens = torch.tensor([20, 0, 0], dtype=torch.int32, device=DEV)
    assert pool.reserve(lens).item() == 1
    i = torch.tensor([0], dtype=torch.int32, device=DEV)
    assert pool.fork(i, i + 1).item() == 1
    new = torch.tensor([1, 1, 0], dtype=torch.int32, device=DEV)
    ctx = pool.lens.clone()
    assert pool.reserve(ctx + 5 * new).item() == 0             # needs a page more than there are
    assert pool.step_rows(ctx, new, 4)[3].tolist() == [-1] * 4
    assert pool.reserve(ctx + new).item() == 1
    cu, seq, pos, slots = pool.step_rows(ctx, new, 4)
    assert cu.tolist() == [0, 1, 2, 2] and seq.tolist() == [0, 1, -1, -1] and pos.tolist() == [20, 20, -1, -1]
    t = pool.table.tolist()
    assert slots.tolist() == [t[0][2] * 8 + 4, t[1][2] * 8 + 4, -1, -1] and t[0][2] != t[1][2]


def test_in_a_graph():
    rng = random.Random(2)
    table = torch.tensor([[rng.randrange(60) for _ in range(9)] for _ in range(6)], dtype=torch.int32, device=DEV)
    ctx = torch.zeros(6, dtype=torch.int32, device=DEV)
    new = torch.tensor([1, 0, 4, 2, 1, 3], dtype=torch.int32, device=DEV)
    kv_pages.step_rows(table, ctx, new, 16, 60, 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_pages.step_rows(table, ctx, new, 16, 60, 16)
    for _ in range(3):
        ctx.add_(new)
        new.copy_(new.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        want = kv_pages.step_rows(table, ctx, new, 16, 60, 16)
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        assert [x.tolist() for x in out] == list(_lists(table.tolist(), ctx.tolist(), new.tolist(), 16, 60, 16))
