"""Tree steps whose room was refused (pool.reserve gave ok 0): nothing of the pool, the caches, the
block summaries or the contexts changes, and the next step finds everything as it was."""

import math

import pytest
import torch

from ananta_ocr_amd import kv_pages, pipeline, tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
IDX = 128.0 / math.sqrt(128.0)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("width", [128, 64])
@pytest.mark.parametrize("captured", [False, True])
def test_a_refused_step_changes_nothing(width, captured):
    """Row 3 holds the pages that the step needs, or does not: the same calls, eager or one graph."""
    bs, H, V, B, pages = 64, 2, 500, 4, 20
    g = torch.Generator().manual_seed(width)
    k, v = (torch.randn(pages, bs, H, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    ik, hc = torch.randn(pages, bs, width, generator=g).to(DEV), torch.randn(width, generator=g).to(DEV)
    state = pipeline.KBarPageCache(pages, width, DEV)
    pool = kv_pages.PagePool(kv_pages.PageCaches([k, v, ik], pages=[state.kbar]), B, 9)
    nodes = [9, 6, 1, 0]
    T = sum(nodes)
    start = _i32([4 * bs + 60, 3 * bs, 5, 0])            # the first two need a page more, the third none
    cu = _i32([0] + nodes).cumsum(0).to(torch.int32)
    room = start + _i32(nodes)
    held = [pool.refs, pool.table, pool.lens, k, v, ik, state.kbar]
    states = {}
    for hog in (0, 9 * bs, 8 * bs):                     # 9 + 9 pages and two more, 9 + 8 and three
        pool.free(torch.zeros_like(start))
        lens = start.clone()
        lens[3] = hog
        assert int(pool.reserve(lens)) == 1
        if hog == 9 * bs:                               # two pages left, of which one is taken
            pool.refs[torch.nonzero(pool.refs == 0)[0]] = 1
        state.put_sequences(ik, hc, bs, pool.table.clamp(min=0), pool.lens)
        states[hog] = [x.clone() for x in held]
    ctx = start.clone()
    ctx[3] = 0
    q, iq = torch.zeros(T, H, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(T, width, device=DEV)
    score, tokens, parents = torch.zeros(T, V, device=DEV), _i32([0] * T), _i32([0] * T)

    def fill(seed, hog):
        g = torch.Generator().manual_seed(seed)
        par = [x for n in nodes for x in ([-1] + [int(torch.randint(0, i, (1,), generator=g))
                                                 for i in range(1, n)])[:n]]
        for x, y in ((q, torch.randn(T, H, 128, generator=g)), (iq, torch.randn(T, width, generator=g)),
                     (score, torch.randn(T, V, generator=g)), (parents, torch.tensor(par)),
                     (tokens, torch.randint(0, V, (T,), generator=g))):
            x.copy_(y)
        o = 0
        for n in nodes:                                 # the last node's chain is accepted
            i = n - 1
            while i > 0:
                score[o + par[o + i], tokens[o + i].long()] = 9.0 + 0.1 * i
                i = par[o + i]
            o += n
        for x, y in zip(held, states[hog]):
            x.copy_(y)

    def step():
        ok = pool.reserve(room)
        out = pipeline.tree_step(state, q, k, v, iq, bs, 1, IDX, 1e-4, 1.0, 3, 4, pool.table, ctx, cu,
                                 parents, max(nodes))
        found = tree.verify_tree(score, tokens, parents, cu, max(nodes))
        new = pipeline.commit_tree(pool, found[1], found[0], ctx, [(state, ik, hc)])
        return [ok, out, *found, new]

    fill(0, 0)
    run = step
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()

        def run():
            graph.replay()
            return kept
    for seed, hog in ((1, 0), (2, 9 * bs), (3, 8 * bs), (4, 9 * bs), (5, 0)):
        fill(seed, hog)
        ok, _, count, path, _, new = run()
        torch.cuda.synchronize()
        assert int(ok) == (hog != 9 * bs), hog
        assert int(count[0]) > 1 and int(count[2]) == 1
        if hog == 9 * bs:
            # the requests that lack their slots stay, the others (none here: all or no rows) too
            assert torch.equal(new, ctx)
            for x, y in zip(held, states[hog]):
                assert torch.equal(x, y)
        else:
            assert new.tolist() == [int(a) + int(b) for a, b in zip(ctx, count)]
            assert pool.lens.tolist()[:3] == new.tolist()[:3]


def test_rows_that_hold_some_of_their_nodes():
    """Only where a row holds the slot of its last accepted node do its nodes stand, whatever it
    holds of the others."""
    bs = 4
    x = torch.arange(12 * bs, dtype=torch.float32, device=DEV).view(12, bs, 1).clone()
    pool = kv_pages.PagePool(kv_pages.PageCaches([x]), 5, 4)
    assert int(pool.reserve(_i32([9, 9, 6, 0, 8]))) == 1
    table, lens, old = pool.table.clone(), pool.lens.clone(), x.clone()
    ctx = torch.tensor([5, 5, 6, 0, 5], device=DEV)
    path = torch.tensor([[0, 2, 3], [0, 2, 4], [0, 1, -1], [0, -1, -1], [-1, -1, -1]], device=DEV)
    kept = pool.keep(path, torch.tensor([3, 3, 2, 1, 0], device=DEV), ctx)
    assert kept.tolist() == pool.lens.tolist() == [8, 9, 6, 0, 8]
    assert torch.equal(pool.table[1:], table[1:])
    row = lambda t, r, i: float(t[int(table[r, i // bs]), i % bs, 0])
    assert [row(x, 0, i) for i in range(8)] == [row(old, 0, i) for i in (0, 1, 2, 3, 4, 5, 7, 8)]
    for r in range(1, 5):
        assert [row(x, r, i) for i in range(int(lens[r]))] == [row(old, r, i) for i in range(int(lens[r]))]
    # path entries past count are not looked at
    again = pool.keep(torch.tensor([[0, 7]] * 5, device=DEV), torch.ones(5, dtype=torch.int32, device=DEV),
                      torch.tensor([7, 8, 6, 0, -3], device=DEV))
    assert again.tolist() == [8, 9, 6, 0, 8]


@pytest.mark.parametrize("rows,n", [(1, 1), (255, 3), (256, 4), (1500, 9), (8192, 2)])
def test_what_a_step_leaves_of_many_rows(rows, n):
    """Lengths, contexts and counts of any number of rows against lists; counts past the path and below
    0, contexts below 0, lengths that reach 2^31 - 1."""
    g = torch.Generator().manual_seed(rows)
    rnd = lambda lo, hi: torch.randint(lo, hi, (rows,), generator=g)
    big = 2 ** 31 - 1
    ctx = torch.where(rnd(0, 9) == 0, rnd(-3, 2), rnd(0, 40))
    ctx = torch.where(rnd(0, 9) == 0, big - rnd(0, 4), ctx)
    lens = (ctx + rnd(-2, 2 * n)).clamp(0, big)
    count = rnd(-1, n + 3)
    path = torch.stack([torch.arange(n)] * rows) + torch.randint(0, 2, (rows, n), generator=g).cumsum(1)
    path[:, 0] = 0
    got = kv_pages._keep_lens(path.to(DEV), count.to(DEV), ctx.to(DEV), lens.to(torch.int32).to(DEV))
    want = []
    for p, c, x, m in zip(path.tolist(), count.tolist(), ctx.tolist(), lens.tolist()):
        k = min(c, n)
        ok = k > 0 and x >= 0 and x + p[k - 1] < m
        want.append((k if ok else 0, x + k if ok else m, x + k if ok else x, x + k if ok else 0))
    assert list(zip(*(t.tolist() for t in got))) == want
