"""Speculative steps as a serving loop runs them: tree_step, verify_tree, commit_tree over one
pool, against the same tokens decoded as chunks of known ones (extend_prefill)."""

import math

import pytest
import torch

from ananta_ocr_amd import kv_pages, pipeline, tree
from tree_oracle import ancestors

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 1.0 / math.sqrt(128)
IDX = 128.0 / math.sqrt(128.0)


class Model:
    """q, k, v, index query and key of a token, from its id and position alone: what a tree's node
    and the same token in a chunk have in common."""

    def __init__(self, H, Hkv, V, seed):
        g = torch.Generator().manual_seed(seed)
        self.e = [torch.randn(V, n, 128, generator=g).to(DEV) for n in (H, Hkv, Hkv, 1, 1)]
        self.rot = torch.randn(4096, 128, generator=g).to(DEV) * 0.5

    def __call__(self, ids, pos):
        q, k, v, iq, ik = ((e[ids] + self.rot[pos][:, None]) * 0.6 for e in self.e)
        return q.bfloat16(), k.bfloat16(), v.bfloat16(), iq[:, 0], ik[:, 0]


def _write(caches, table, row, slots, k, v, ik):
    bs = caches[0].shape[1]
    pages = table[row, slots // bs].long()
    for c, x in zip(caches, (k, v, ik)):
        c[pages, slots % bs] = x


def _new(rows, width, H, bs, num_pages):
    k = torch.zeros(num_pages, bs, H, 128, dtype=torch.bfloat16, device=DEV)
    v, ik = torch.zeros_like(k), torch.zeros(num_pages, bs, 128, device=DEV)
    state = pipeline.KBarPageCache(num_pages, 128, DEV)
    pool = kv_pages.PagePool(kv_pages.PageCaches([k, v, ik], pages=[state.kbar]), rows, width)
    return pool, (k, v, ik), state


def _prefill(m, pool, caches, state, hc, prompts, bs):
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=DEV)
    assert int(pool.reserve(lens)) == 1
    for b, ids in enumerate(prompts):
        pos = torch.arange(len(ids), device=DEV)
        _, k, v, _, ik = m(torch.tensor(ids, dtype=torch.long, device=DEV), pos)
        _write(caches, pool.table, b, pos, k, v, ik)
    state.put_sequences(caches[2], hc, bs, pool.table.clamp(min=0), lens)
    return lens


@pytest.mark.parametrize("Hkv,bs,lb,K,topm", [(2, 64, 2, 4, 8), (1, 32, 4, 12, 16)])
def test_loop_equals_chunks(Hkv, bs, lb, K, topm):
    """Four steps of two requests: every accepted node's output, routing and the committed cache
    are those of a second pool that gets the accepted tokens as chunks."""
    H, V, rows = 2, 50, 3
    m = Model(H, Hkv, V, bs)
    g = torch.Generator().manual_seed(bs + 1)
    hc = (torch.randn(128, generator=g) * 0.3).to(DEV)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (bs * 9 + bs - 3, 3 * bs)]
    prompts.append([])                                         # an idle row
    pool, caches, state = _new(rows, 24, Hkv, bs, 60)
    ctx = _prefill(m, pool, caches, state, hc, prompts, bs)
    pool2, caches2, state2 = _new(rows, 24, Hkv, bs, 60)
    _prefill(m, pool2, caches2, state2, hc, prompts, bs)
    args = (bs, lb, IDX, 1e-4, 1.0, K, topm)
    text = [list(p) for p in prompts]
    roots = [7, 8]
    grew = 0
    for it in range(4):
        nodes = [9, 1 + 4 * it, 0]
        par = [[-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, n)]
               if n else [] for n in nodes]
        tok = [[roots[b]] + torch.randint(0, V, (n - 1,), generator=g).tolist() if n else []
               for b, n in enumerate(nodes)]
        cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32).to(DEV)
        room = ctx + torch.tensor(nodes, dtype=torch.int32, device=DEV)
        assert int(pool.reserve(room)) == 1
        qs, iqs = [], []
        for b in range(2):
            c = int(ctx[b])
            dep = torch.tensor([len(ancestors(par[b], i)) - 1 for i in range(nodes[b])], device=DEV)
            q, k, v, iq, ik = m(torch.tensor(tok[b], device=DEV), c + dep)
            _write(caches, pool.table, b, c + torch.arange(nodes[b], device=DEV), k, v, ik)
            qs.append(q)
            iqs.append(iq)
        parents = torch.tensor(sum(par, []), dtype=torch.int32, device=DEV)
        out, (idx, bias, valid), q_pos = pipeline.tree_step(
            state, torch.cat(qs), caches[0], caches[1], torch.cat(iqs), *args, pool.table, ctx, cu,
            parents, max(nodes), out_dtype=torch.float32, return_routing=True)
        # the target: after every node of the deepest chain its child, elsewhere a token of its own
        T = sum(nodes)
        target = torch.rand(T, V, generator=g) * 0.5
        for b in range(2):
            deep = max(range(nodes[b]), key=lambda i: len(ancestors(par[b], i)))
            for child in ancestors(par[b], deep)[:-1]:
                target[int(cu[b]) + par[b][child], tok[b][child]] = 1.0
        tokens = torch.tensor(sum(tok, []), device=DEV)
        count, path, nxt = tree.verify_tree(target.to(DEV), tokens, parents, cu, max(nodes))
        old = ctx
        ctx = pipeline.commit_tree(pool, path, count, ctx, [(state, caches[2], hc)])
        assert ctx.tolist() == [int(old[b]) + int(count[b]) for b in range(3)]
        assert pool.lens.tolist() == ctx.tolist()
        assert int((pool.refs > 0).sum()) == sum(-(-n // bs) for n in ctx.tolist())
        grew += int(count.sum()) - 2
        # the same tokens as a chunk of the second pool
        got = [path[b, :int(count[b])].tolist() for b in range(2)]
        assert int(pool2.reserve(ctx)) == 1
        q2, iq2 = [], []
        for b in range(2):
            pos = int(old[b]) + torch.arange(len(got[b]), device=DEV)
            ids = torch.tensor([tok[b][i] for i in got[b]], device=DEV)
            q, k, v, iq, ik = m(ids, pos)
            _write(caches2, pool2.table, b, pos, k, v, ik)
            q2.append(q.repeat_interleave(1, 1))
            iq2.append(iq)
            text[b] += ids.tolist()
        cu2 = torch.tensor([0, len(got[0]), len(got[0]) + len(got[1]), len(got[0]) + len(got[1])],
                           dtype=torch.int32, device=DEV)
        k2, v2 = (x.repeat_interleave(H // Hkv, 2) for x in caches2[:2])
        ref, (idx2, bias2, valid2), pos2 = pipeline.extend_prefill(
            state2, torch.cat(q2), k2, v2, torch.cat(iq2), caches2[2], hc, *args,
            pool2.table.clamp(min=0), ctx, old, cu2, max_query_len=max(map(len, got)),
            out_dtype=torch.float32, return_routing=True)
        at = torch.cat([int(cu[b]) + path[b, :len(got[b])].long() for b in range(2)])
        assert torch.equal(q_pos[at], pos2)
        assert torch.equal(valid[at].bool(), valid2) and torch.equal(
            torch.where(valid2, idx[at], -1), torch.where(valid2, idx2, -1))
        # outputs to the fp32 sums of both (routing biases are the same bits)
        assert float((out[at] - ref).abs().max()) <= 1e-4
        for b in range(2):
            n = int(ctx[b])
            slots = torch.arange(n, device=DEV)
            for x, y in zip(caches, caches2):
                a, c = (t[p.table[b, slots // bs].long(), slots % bs] for t, p in ((x, pool), (y, pool2)))
                assert torch.equal(a, c)
            blocks = torch.arange(-(-n // bs), device=DEV)
            a, c = (s.kbar[p.table[b, blocks].long()] for s, p in ((state, pool), (state2, pool2)))
            assert torch.equal(a, c)
        roots = [int(x) for x in nxt[:2]]
        if it == 1:                                            # moved together in between
            pool.free(torch.where(torch.tensor([1, 1, 0], device=DEV) > 0, ctx, 0))
            pool.compact()
    assert grew > 4


@pytest.mark.parametrize("width", [128, 64])
def test_a_captured_step(width):
    """Reserve, attention, verification and commit in one graph: every replay gives what the same
    calls give outside of it, on other inputs and after other work."""
    bs, H, V, B = 64, 2, 3000, 3
    g = torch.Generator().manual_seed(width)
    k, v = (torch.randn(30, bs, H, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    ik, hc = torch.randn(30, bs, width, generator=g).to(DEV), torch.randn(width, generator=g).to(DEV)
    state = pipeline.KBarPageCache(30, width, DEV)
    pool = kv_pages.PagePool(kv_pages.PageCaches([k, v, ik], pages=[state.kbar]), B, 9)
    start = torch.tensor([5 * bs + 60, 3 * bs, 0], dtype=torch.int32, device=DEV)
    assert int(pool.reserve(start)) == 1
    state.put_sequences(ik, hc, bs, pool.table.clamp(min=0), start)
    nodes = [7, 5, 1]
    T = sum(nodes)
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32).to(DEV)
    room = start + cu[1:] - cu[:-1]
    held = [pool.refs, pool.table, pool.lens, k, v, ik, state.kbar]
    before = [x.clone() for x in held]
    q = torch.zeros(T, H, 128, dtype=torch.bfloat16, device=DEV)
    iq, u = torch.zeros(T, width, device=DEV), torch.zeros(T, device=DEV)
    probs, draft = torch.full((T, V), 1.0 / V, device=DEV), torch.full((T, V), 1.0 / V, device=DEV)
    tokens, parents = (torch.zeros(T, dtype=torch.int32, device=DEV) for _ in range(2))

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        logits = torch.randn(T, V, generator=g) * 3
        p, d = logits.softmax(-1), (logits + torch.randn(T, V, generator=g) * 0.3).softmax(-1)
        par = [x for n in nodes for x in [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)]]
        first = [c for c, n in zip(cu.tolist(), nodes) for _ in range(n)]
        at = torch.tensor([f + max(x, 0) for f, x in zip(first, par)])
        for x, y in ((q, torch.randn(T, H, 128, generator=g)), (iq, torch.randn(T, width, generator=g)),
                     (u, torch.rand(T, generator=g)), (probs, p), (draft, d),
                     (parents, torch.tensor(par)),
                     (tokens, torch.multinomial(d[at], 1, generator=g)[:, 0])):
            x.copy_(y)
        for x, y in zip(held, before):
            x.copy_(y)

    def step():
        ok = pool.reserve(room)
        out = pipeline.tree_step(state, q, k, v, iq, bs, 2, IDX, 1e-4, 1.0, 3, 4, pool.table, start, cu,
                                 parents, 7)
        found = tree.verify_tree(probs, tokens, parents, cu, 7, uniforms=u, draft=draft)
        new = pipeline.commit_tree(pool, found[1], found[0], start, [(state, ik, hc)])
        return [ok, out, *found, new]
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    counts = set()
    for seed in range(1, 7):
        fill(seed)
        want = [x.clone() for x in (*step(), *held)]
        (q.float() @ q.float().transpose(1, 2)).sum()         # other work between
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, (*kept, *held)))
        counts.add(tuple(want[2].tolist()))
    assert len(counts) > 1


def test_forked_requests_decode_apart():
    """A request forked to two rows, each grown by a tree of its own: both read the shared pages and
    their own copy of the last one, and the first row's outputs are what they were."""
    bs, H, V = 64, 2, 40
    m = Model(H, H, V, 3)
    g = torch.Generator().manual_seed(2)
    hc = torch.zeros(128, device=DEV)
    pool, caches, state = _new(3, 12, H, bs, 40)
    prompt = torch.randint(0, V, (bs * 5 + 20,), generator=g).tolist()
    _prefill(m, pool, caches, state, hc, [prompt, [], []], bs)
    args = (bs, 1, IDX, 1e-4, 1.0, 4, 8)
    n0 = len(prompt)

    def step(rows, toks):
        ctx = torch.full((len(rows),), n0, dtype=torch.int32, device=DEV)
        room = pool.lens.clone()
        for r in rows:
            room[r] = n0 + 4
        assert int(pool.reserve(room)) == 1
        par = [-1, 0, 0, 1]
        dep = torch.tensor([0, 1, 1, 2], device=DEV)
        qs = []
        for r, t in zip(rows, toks):
            q, k, v, iq, ik = m(torch.tensor(t, device=DEV), n0 + dep)
            _write(caches, pool.table, r, n0 + torch.arange(4, device=DEV), k, v, ik)
            qs.append((q, iq))
        cu = torch.arange(len(rows) + 1, dtype=torch.int32, device=DEV) * 4
        return pipeline.tree_step(state, torch.cat([a for a, _ in qs]), *caches[:2],
                                  torch.cat([b for _, b in qs]), *args, pool.table[rows], ctx, cu,
                                  torch.tensor(par * len(rows), dtype=torch.int32, device=DEV), 4,
                                  out_dtype=torch.float32)
    assert int(pool.fork(torch.tensor([0, 0], device=DEV), torch.tensor([1, 2], device=DEV))) == 1
    toks = [[1, 2, 3, 4], [5, 6, 7, 8], [9, 10, 11, 12]]
    all3 = step([0, 1, 2], toks)
    assert int(pool.refs.max()) == 3
    for r in range(3):
        one = step([r], [toks[r]])
        assert float((all3[4 * r:4 * r + 4] - one).abs().max()) <= 1e-4
    # the children leave: the first row's pages are its own again
    pool.free(torch.tensor([n0, 0, 0], device=DEV))
    assert pool.refs.max() == 1 and int((pool.refs > 0).sum()) == -(-n0 // bs)
    assert float((step([0], [toks[0]]) - all3[:4]).abs().max()) <= 1e-4


@pytest.mark.parametrize("width", [128, 64])
def test_padded_and_empty_batches(width):
    """Rows past the last tree, as a batch of fixed size has them, change nothing; nor do no rows at
    all fail."""
    bs, H = 64, 2
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(12, bs, H, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    ik, hc = torch.randn(12, bs, width, generator=g).to(DEV), torch.randn(width, generator=g).to(DEV)
    table = torch.randperm(12, generator=g).to(torch.int32).view(2, 6).to(DEV)
    ctx = torch.tensor([5 * bs + 3, 4 * bs], dtype=torch.int32, device=DEV)
    state = pipeline.KBarPageCache(12, width, DEV)
    state.put_sequences(ik, hc, bs, table, ctx)
    q, iq = torch.randn(40, H, 128, generator=g).bfloat16().to(DEV), torch.randn(40, width, generator=g).to(DEV)
    par = torch.randint(-3, 40, (40,), generator=g).to(torch.int32).to(DEV)
    cu = torch.tensor([0, 6, 10], dtype=torch.int32, device=DEV)
    call = lambda n, cu, most: pipeline.tree_step(state, q[:n], k, v, iq[:n], bs, 1, IDX, 1e-4, 1.0, 3, 4, table,
                                                  ctx, cu, par[:n], most, out_dtype=torch.float32)
    want = call(10, cu, 6)
    for _ in range(3):
        torch.full((4096,), -1, dtype=torch.int32, device=DEV)          # memory that held something
        assert torch.equal(call(40, cu, 6)[:10], want)
    assert call(0, torch.zeros_like(cu), 0).shape == (0, H, 128)


@pytest.mark.parametrize("width", [128, 64])
def test_requests_that_stay_leave_shared_pages_alone(width):
    """Row 1 shares its pages with row 0 and is cut inside one; while row 0 takes a step, row 1's
    summaries are not recomputed, and the pages that both name keep theirs."""
    bs = 64
    g = torch.Generator().manual_seed(8)
    ik = torch.randn(9, bs, width, generator=g).to(DEV)
    kv = torch.randn(9, bs, 1, 128, generator=g).bfloat16().to(DEV)
    hc = torch.randn(width, generator=g).to(DEV)
    state = pipeline.KBarPageCache(9, width, DEV)
    pool = kv_pages.PagePool(kv_pages.PageCaches([kv, ik], pages=[state.kbar]), 2, 5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    assert int(pool.reserve(i32([3 * bs, 0]))) == 1
    state.put_sequences(ik, hc, bs, pool.table[:1], pool.lens[:1])
    assert int(pool.fork(i32([0]), i32([1]))) == 1
    pool.free(i32([3 * bs, bs + 7]))
    assert int(pool.reserve(i32([3 * bs + 3, 0]))) == 1
    before = state.kbar.clone()
    new = pipeline.commit_tree(pool, i32([[0, 2, -1], [-1, -1, -1]]), i32([2, 0]), i32([3 * bs, bs + 7]),
                               [(state, ik, hc)])
    assert new.tolist() == pool.lens.tolist() == [3 * bs + 2, bs + 7]
    grown = int(pool.table[0, 3])
    keep = [p for p in range(9) if p != grown]
    assert torch.equal(state.kbar[keep], before[keep])
    want = pipeline.KBarPageCache(9, width, DEV)
    want.put_sequences(ik, hc, bs, pool.table[:1], pool.lens[:1])
    assert float((state.kbar[grown] - want.kbar[grown]).abs().max()) <= 1e-5


def test_index_keys_of_another_width_and_requests_without_context():
    """Index queries of 64 dims (the general scores), and a request whose tree is all there is: a chain
    gives extend_prefill's rows, a row without committed blocks routes nowhere."""
    bs, H, d = 64, 2, 64
    g = torch.Generator().manual_seed(5)
    ctx, n = [bs * 6 + 9, 0], [5, 4]
    pages = [-(-(c + m) // bs) for c, m in zip(ctx, n)]
    table = torch.zeros(2, max(pages), dtype=torch.int32)
    perm = torch.randperm(12, generator=g)
    table[0, :pages[0]], table[1, 0] = perm[:pages[0]].int(), perm[-1].int()
    k, v = (torch.randn(12, bs, H, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    for width in (d, 128):
        ik = torch.randn(12, bs, width, generator=g).to(DEV)
        hc = torch.randn(width, generator=g).to(DEV) * 0.2
        q = torch.randn(9, H, 128, generator=g).bfloat16().to(DEV)
        iq = torch.randn(9, width, generator=g).to(DEV)
        t, c = table.to(DEV), torch.tensor(ctx, device=DEV)
        cu = torch.tensor([0, 5, 9], device=DEV)
        args = (bs, 2, IDX, 1e-4, 1.0, 3, 4)
        state = pipeline.KBarPageCache(12, width, DEV)
        state.put_sequences(ik, hc, bs, t, c)
        par = torch.tensor([-1, 0, 1, 2, 3, -1, 0, 1, 2], device=DEV)
        out, (idx, bias, valid), pos = pipeline.tree_step(
            state, q, k, v, iq, *args, t, c, cu, par, 5, out_dtype=torch.float32, return_routing=True)
        assert pos.tolist() == [393, 394, 395, 396, 397, 0, 1, 2, 3]
        assert bool(valid[:5].any()) and not bool(valid[5:].any())
        ref, (idx2, _, valid2), _ = pipeline.extend_prefill(
            state, q, k, v, iq, ik, hc, *args, t, c + torch.tensor(n, device=DEV), c, cu,
            max_query_len=5, out_dtype=torch.float32, return_routing=True)
        assert torch.equal(valid[:5].bool(), valid2[:5])
        assert torch.equal(torch.where(valid2[:5], idx[:5], -1), torch.where(valid2[:5], idx2[:5], -1))
        assert float((out - ref).abs().max()) <= 1e-4
