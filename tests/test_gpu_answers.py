"""Several answers to shared prompts, the operators together as a serving loop runs them: prompts in the
pool's pages, rows forked, and step after step the new tokens' slots, their rotated keys and values
written, attention that reads the prompts once, and the next tokens drawn.  Against 64 bits, sequence by
sequence.

Tolerance: a key in the cache is the rotated one rounded to bf16, and the reference rounds its own the same
way but for roundings of 6 2^-24 before it, which may fall to either side: such a key is off by a step, 2^-8
of its value of up to 3, in one of 128 products with a query of about 1, a score by 1e-3 (3 * 2^-8 / 11.3).
Few fall so (one in 2^14), none twice in a score as a rule: a weight is off by 1e-3 of itself and an output
by 1e-3 of the largest |v|, 5, beside the half step of bf16, 2^-8 of its value: 6e-3 + 2^-8 |o| + 1e-3."""

import math

import pytest
import torch

from ananta_ocr_amd import kv_pages, pipeline, rope, sampling

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32
H, HKV, D, V = 4, 2, 128, 500


def _turned(x, pos, f):
    """bf16 [n, heads, D] rotated in 64 bits, halves, rounded to bf16."""
    a = pos.double()[:, None, None] * f
    u, v = x.double()[..., :D // 2], x.double()[..., D // 2:]
    return torch.cat((u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()), -1).bfloat16()


class _Serving:
    def __init__(self, page, rows, pages, layers, seed):
        g = torch.Generator().manual_seed(seed)
        self.g, self.rows = g, rows
        self.k = torch.zeros(layers, pages, page, HKV, D, device=DEV).bfloat16()
        self.v = torch.zeros_like(self.k)
        self.pool = kv_pages.PagePool(kv_pages.PageCaches([self.k, self.v], layered=True), rows, 40)
        self.f, _ = rope.inv_freq(D, device=DEV)
        self.head = (torch.randn(H * D, V, generator=g) * 0.05).to(DEV)
        self.keys = [[[] for _ in range(rows)] for _ in range(layers)]     # what every row's tokens hold

    def qkv(self, T):
        return [[torch.randn(T, n, D, generator=self.g).bfloat16().to(DEV) for n in (H, HKV, HKV)]
                for _ in range(len(self.k))]

    def step(self, new, qkv, groups, prefix, T):
        st = pipeline.start_step(self.pool, torch.tensor(new, dtype=I32, device=DEV), T)
        return st, [pipeline.shared_step(st, *x, self.k[l], self.v[l], self.pool.table, self.f, groups, prefix)
                    for l, x in enumerate(qkv)]

    def reference(self, new, ctx, qkv):
        """Outputs in 64 bits; the rows' keys and values grow by the step's."""
        outs = []
        for l, (q, k, v) in enumerate(qkv):
            r, rows = 0, []
            for b, n in enumerate(new):
                pos = ctx[b] + torch.arange(n, device=DEV)
                mine = self.keys[l][b]
                mine.append((_turned(k[r:r + n], pos, self.f), v[r:r + n].clone()))    # (v is written again)
                ks, vs = (torch.cat([x[i] for x in mine]).double().repeat_interleave(H // HKV, 1) for i in (0, 1))
                qq = _turned(q[r:r + n], pos, self.f).double()
                for i in range(n):
                    m = ctx[b] + i + 1
                    z = (qq[i][:, None] * ks[:m].transpose(0, 1)).sum(-1) / math.sqrt(D)
                    rows.append((torch.softmax(z, -1)[..., None] * vs[:m].transpose(0, 1)).sum(1))
                r += n
            outs.append(torch.stack(rows) if rows else torch.zeros(0, H, D, device=DEV).double())
        return outs


def _close(out, ref):
    assert out.dtype == torch.bfloat16
    err = (out[:len(ref)].double() - ref).abs()
    assert bool((err <= 7e-3 + 2.0 ** -8 * ref.abs()).all()), err.max().item()
    assert not out[len(ref):].any()


@pytest.mark.parametrize("page", [16, 7, 64])
def test_answers_step_by_step(page):
    """Two prompts, forked into three and two answers, five steps of one to three tokens each; one answer
    pauses, one leaves, tokens drawn from the outputs."""
    s = _Serving(page, 7, 200, 2, page)
    prompts = [83, 40]
    new = prompts + [0] * 5
    qkv = s.qkv(sum(new) + 2)
    _, outs = s.step(new, qkv, None, None, sum(new) + 2)
    for o, r in zip(outs, s.reference(new, [0] * 7, qkv)):
        _close(o, r)
    src = torch.tensor([0, 0, 0, 1, 1], dtype=I32, device=DEV)
    assert s.pool.fork(src, torch.arange(2, 7, dtype=I32, device=DEV)).item() == 1
    for l in range(2):
        for b, a in zip(range(2, 7), [0, 0, 0, 1, 1]):
            s.keys[l][b] = list(s.keys[l][a])
    # the pool's rows: 0 and 1 the prompts, then the answers of each
    groups = torch.tensor([2, 5, 7], dtype=I32, device=DEV)
    prefix = torch.tensor([p // page * page for p in prompts], dtype=I32, device=DEV)
    lens = prompts + [83] * 3 + [40] * 2
    shared_pages = s.pool.table[2, :83 // page]
    assert torch.equal(shared_pages, s.pool.table[0, :83 // page])
    for t, new in enumerate(([0, 0, 1, 1, 1, 1, 1], [0, 0, 1, 3, 1, 0, 2], [0, 0, 2, 1, 1, 1, 1],
                             [0, 0, 1, 1, 0, 1, 1], [0, 0, 3, 2, 0, 1, 1])):
        if t == 3:                               # an answer leaves
            keep = s.pool.lens.clone()
            keep[4] = 0
            s.pool.free(keep)
            lens[4] = 0
        T = sum(new) + t % 2
        qkv = s.qkv(T)
        st, outs = s.step(new, qkv, groups, prefix, T)
        assert st.ok.item() == 1 and st.context_lens.tolist() == lens
        for o, r in zip(outs, s.reference(new, lens, qkv)):
            _close(o, r)
        lens = [a + b for a, b in zip(lens, new)]
        assert s.pool.lens.tolist() == lens
        # the last row of every sequence draws its next token
        last = (st.cu_seqlens_q[1:] - 1).long()[[b for b in range(7) if new[b]]]
        logits = outs[-1].float().reshape(T, -1)[last] @ s.head
        u = torch.rand(len(last), generator=s.g).to(DEV)
        token, probs = sampling.sample(logits, u, 0.8, 40, 0.95, return_probs=True)
        assert bool((probs.gather(1, token[:, None]) > 0).all()) and bool(((probs > 0).sum(1) <= 40).all())
        run = probs.double().cumsum(1)
        before = run.gather(1, token[:, None])[:, 0] - probs.double().gather(1, token[:, None])[:, 0]
        upto = run.gather(1, token[:, None])[:, 0]
        # (probabilities in fp32: a sum of up to 40 is off by 40 2^-25)
        assert bool((before <= u.double() + 2e-6).all()) and bool((upto >= u.double() - 2e-6).all())


def test_a_refused_step_writes_nothing():
    s = _Serving(8, 3, 5, 1, 3)          # 3 pages, a copy of the last, and one of the two that growth takes
    new = [20, 0, 0]
    qkv = s.qkv(20)
    s.step(new, qkv, None, None, 20)
    assert s.pool.fork(torch.tensor([0], dtype=I32, device=DEV), torch.tensor([1], dtype=I32, device=DEV)).item()
    before = s.k.clone(), s.v.clone(), s.pool.table.clone(), s.pool.refs.clone(), s.pool.lens.clone()
    st, _ = s.step([9, 9, 0], s.qkv(18), None, None, 18)
    assert st.ok.item() == 0 and st.slots.tolist() == [-1] * 18
    after = s.k, s.v, s.pool.table, s.pool.refs, s.pool.lens
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_step_in_a_graph():
    """A whole step of a batch of a fixed size captured: room, slots, keys, attention, tokens.  Replays,
    with eager reads of the pool between them, against 64 bits."""
    s = _Serving(16, 5, 120, 2, 9)
    new = [50, 0, 0, 0, 0]
    qkv = s.qkv(50)
    s.step(new, qkv, None, None, 50)
    s.reference(new, [0] * 5, qkv)
    assert s.pool.fork(torch.zeros(4, dtype=I32, device=DEV), torch.arange(1, 5, dtype=I32, device=DEV)).item() == 1
    for l in range(2):
        for b in range(1, 5):
            s.keys[l][b] = list(s.keys[l][0])
    T = 8
    n = torch.zeros(5, dtype=I32, device=DEV)                # (no new token: the capture's warm-up)
    buf = s.qkv(T)
    groups, prefix = torch.tensor([0, 5], dtype=I32, device=DEV), torch.tensor([48], dtype=I32, device=DEV)
    u = torch.zeros(T, device=DEV)

    def run():
        st = pipeline.start_step(s.pool, n, T)
        outs = [pipeline.shared_step(st, *x, s.k[l], s.v[l], s.pool.table, s.f, groups, prefix)
                for l, x in enumerate(buf)]
        logits = outs[-1].float().reshape(T, -1) @ s.head
        return st, outs, sampling.sample(logits, u, 0.9, 20, 0.9), logits

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st, outs, token, logits = run()
    lens = [50] * 5
    assert s.pool.lens.tolist() == lens
    for i, new in enumerate(([0, 1, 1, 1, 1], [0, 2, 1, 1, 1], [1, 1, 0, 3, 1], [0, 0, 0, 0, 1])):
        n.copy_(torch.tensor(new, dtype=I32))
        for x, y in zip(buf, s.qkv(T)):
            for a, b in zip(x, y):
                a.copy_(b)
        u.copy_(torch.rand(T, generator=s.g))
        graph.replay()
        torch.cuda.synchronize()
        assert st.ok.item() == 1
        for o, r in zip(outs, s.reference(new, lens, buf)):
            _close(o, r)
        assert torch.equal(token, sampling.sample(logits, u, 0.9, 20, 0.9))
        lens = [a + b for a, b in zip(lens, new)]
        assert s.pool.lens.tolist() == lens
