"""Verification of drafted tokens (tree.verify_tree) against a walk in plain Python with 64-bit
sums: paths, counts and drawn tokens are whole numbers and have to be equal."""

import math

import pytest
import torch

from ananta_ocr_amd import tree
from tree_oracle import verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(nodes, V, mode, dtype, seed, siblings=4):
    g = torch.Generator().manual_seed(seed)
    T = sum(nodes)
    logits = torch.randn(T, V, generator=g) * 2.5
    q = torch.softmax(logits + 0.8 * torch.randn(T, V, generator=g), -1)
    p = torch.softmax(logits, -1).to(dtype)
    par, tokens, r = [], [], 0
    for n in nodes:
        own = [-1][:n] + [i - 1 if mode == "chain" else (i - 1) // siblings for i in range(1, n)]
        par.append(own)
        for i in range(n):
            row = q[r + max(own[i], 0)]
            rank = sum(own[j] == own[i] for j in range(i))
            tokens.append(int(torch.multinomial(row, 1, generator=g)) if mode in ("chain", "drawn")
                          else int(row.topk(min(V, rank + 1)).indices[-1]))
        r += n
    u = torch.rand(T, generator=g)
    draft = q.to(dtype) if mode in ("chain", "drawn") else None
    if mode == "greedy":
        p, u = logits.to(dtype), None
    return p, tokens, par, u, draft, nodes


def _check(p, tokens, par, u, draft, nodes, tok_type=torch.int64, view=lambda x: x):
    cu = torch.tensor([0] + nodes).cumsum(0)
    n = max(nodes + [0])
    d = [None if x is None else view(x.to(DEV)) for x in (p, draft)]
    count, path, token = tree.verify_tree(
        d[0], torch.tensor(tokens, dtype=tok_type).to(DEV),
        torch.tensor(sum(par, []), dtype=torch.int32).to(DEV), cu.to(torch.int32).to(DEV), n,
        uniforms=None if u is None else u.to(DEV), draft=d[1])
    assert count.dtype == path.dtype == torch.int32 and token.dtype == torch.int64
    count, path, token = count.tolist(), path.tolist(), token.tolist()
    for b, m in enumerate(nodes):
        r = slice(int(cu[b]), int(cu[b + 1]))
        want, nxt = verify(p[r], tokens[r], par[b], None if u is None else u[r],
                           None if draft is None else draft[r])
        assert count[b] == len(want), (b, count[b], want)
        assert path[b] == want + [-1] * (n - len(want)), b
        assert token[b] == nxt, (b, token[b], nxt)
    return count


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mode", ["chain", "drawn", "best", "greedy"])
@pytest.mark.parametrize("nodes,V", [([6], 1000), ([1, 17, 0, 40], 4097), ([9] * 30, 37),
                                     ([3, 256], 20011)])
def test_walks(mode, nodes, V, dtype):
    total = []
    for seed in range(3):
        total += _check(*_case(nodes, V, mode, dtype, seed), tok_type=(torch.int64, torch.int32)[seed % 2])
    if len(nodes) > 10:
        assert max(total) > 2 and min(total) < max(total)      # drafts stood, and did not


@pytest.mark.parametrize("mode", ["chain", "drawn", "best", "greedy"])
def test_many_vocabularies(mode):
    """One token, around the pieces' borders, and a large odd one."""
    for V in (1, 2, 4095, 4096, 8192, 8193, 131073):
        _check(*_case([5, 2], V, mode, torch.float32, V))


def test_rows_of_a_wider_tensor():
    """Rows that start off a 16-byte boundary, rows of odd strides, and a transposed tensor."""
    for mode in ("chain", "greedy"):
        for dtype in (torch.float32, torch.bfloat16):
            c = _case([7, 12], 9001, mode, dtype, 5)

            def odd(x):
                w = torch.zeros(x.shape[0], x.shape[1] + 6, dtype=x.dtype, device=DEV)
                w[:, 3:-3] = x
                return w[:, 3:-3]
            _check(*c, view=odd)
            _check(*c, view=lambda x: x.t().contiguous().t())


def test_borders_of_the_random_numbers():
    """0 accepts whatever has any probability and draws the first token left; just below 1 accepts
    only what is certain and draws the last."""
    for mode in ("chain", "drawn", "best"):
        for value in (0.0, 1.0 - 2.0 ** -24, 1.0):
            p, tokens, par, u, draft, nodes = _case([8, 20], 300, mode, torch.float32, 2)
            _check(p, tokens, par, torch.full_like(u, value), draft, nodes)


def test_what_is_left_of_a_row():
    V = 6
    one = [[-1, 0, 0]]
    p = torch.zeros(3, V)
    u = torch.tensor([0.5, 0.9, 0.9])
    # both children hold the whole mass and are rejected by their numbers: the last token left
    p[0] = torch.tensor([0.0, 0.5, 0.0, 0.5, 0.0, 0.0])
    _check(p, [0, 1, 3], one, u * 0 + torch.tensor([0.5, 0.9, 1.0]), None, [3])
    # a repeated child's token is gone after its first rejection, an id outside is no token
    p[0] = torch.tensor([0.1, 0.4, 0.1, 0.2, 0.1, 0.1])
    _check(p, [0, 1, 1], one, torch.tensor([0.3, 0.9, 0.0]), None, [3])
    _check(p, [0, -1, V], one, torch.tensor([0.3, 0.0, 0.0]), None, [3])
    _check(p, [0, -1, V], one, torch.tensor([0.3, 0.0, 0.0]), torch.full((3, V), 1 / 6.0), [3])
    # the draft equals the target: what is left is nothing, and the row itself is drawn from
    _check(p, [0, 1, 2], one, torch.tensor([0.3, 1.0, 1.0]), p.clone(), [3])
    # no probability anywhere; values that count as 0
    _check(torch.zeros(3, V), [0, 1, 2], one, u, None, [3])
    p[0] = torch.tensor([math.nan, -1.0, 0.25, math.nan, 0.75, 0.0])
    _check(p, [0, 0, 1], one, u, None, [3])
    # drafted tokens whose draft probability is 0
    q = torch.zeros(3, V)
    q[0, 5] = 1.0
    p[0] = torch.tensor([0.1, 0.4, 0.1, 0.2, 0.2, 0.0])
    _check(p, [0, 5, 1], one, torch.tensor([0.3, 0.5, 0.5]), q, [3])


def test_draft_values_and_numbers_that_count_as_0():
    """NaN and negative draft probabilities neither hold mass back nor add any, and a number below
    0 draws like 0."""
    one = [[-1, 0, 0]]
    p, q = torch.zeros(3, 6), torch.zeros(3, 6)
    p[0] = torch.tensor([0.1, 0.4, 0.1, 0.2, 0.2, 0.0])
    q[0] = torch.tensor([math.nan, 0.8, -0.5, math.nan, 0.2, math.nan])
    for last in (0.0, 0.2, 0.45, 0.75, 0.999):
        # left after token 1: (0.1, 0, 0.1, 0.2, 0, 0); token 0 is then rejected by its number 1
        _check(p, [0, 1, 0], one, torch.tensor([last, 0.9, 1.0]), q, [3])
    _check(p, [0, 5, 3], one, torch.tensor([0.3, 0.0, 0.5]), q, [3])
    below = [[-1, 0]]
    _check(p[:2], [0, 5], below, torch.tensor([0.0, 0.0]), None, [2])
    c = [tree.verify_tree(p[:2].to(DEV), torch.tensor([0, 5], device=DEV),
                          torch.tensor([-1, 0], dtype=torch.int32, device=DEV),
                          torch.tensor([0, 2], dtype=torch.int32, device=DEV), 2,
                          uniforms=torch.tensor([u, u], device=DEV)) for u in (0.0, -0.5, math.nan)]
    for x in c[1:]:
        assert all(torch.equal(s, t) for s, t in zip(c[0], x))


def test_greedy_ties_and_odd_rows():
    V = 20000
    p = torch.zeros(4, V)
    p[0, [77, 15000, 19999]] = 3.0
    p[1] = -math.inf
    p[2] = -math.inf
    p[2, 9] = math.nan
    p[2, 12345] = -5.0
    p[3] = math.nan
    p[3, V - 1] = -math.inf
    par = [[-1, 0, 0, 0]]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check(p.to(dtype), [0, 15000, 77, 77], par, None, None, [4])
    _check(p, [0, 77, 0, 12345], [[-1, 0, 1, 2]], None, None, [4])
    # best tokens past the wavefronts' shares, at every place once
    for at in (0, 63, 64, 255, 256, 8191, 8192, 16383, 19999):
        p = torch.zeros(1, V).bfloat16()
        p[0, at] = 1.0
        _check(p, [0], [[-1]], None, None, [1])


def test_parents_that_are_no_earlier_node():
    p, tokens, par, u, draft, nodes = _case([8], 50, "best", torch.float32, 3)
    par[0] = [3, 0, -1, 7, 1, 1, 99, -5]
    _check(p, tokens, par, u, draft, nodes)


def test_types_that_differ():
    p, tokens, par, u, draft, nodes = _case([9, 9], 777, "drawn", torch.float32, 4)
    half = draft.bfloat16()
    a = [x.to(DEV) for x in (torch.tensor(tokens), torch.tensor(sum(par, [])))]
    cu = torch.tensor([0, 9, 18], device=DEV)
    got = tree.verify_tree(p.to(DEV), *a, cu, 9, uniforms=u.double().to(DEV), draft=half.to(DEV))
    want = tree.verify_tree(p.to(DEV), *a, cu, 9, uniforms=u.to(DEV), draft=half.float().to(DEV))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("mode", ["chain", "drawn", "best"])
def test_first_token_follows_the_target(mode):
    """The token after the root (the first accepted drafted one, else the drawn one) has the
    target's probabilities: over 60,000 sequences each frequency within 5 standard deviations."""
    B, V, m = 60000, 7, 3
    g = torch.Generator(DEV).manual_seed(1)
    row = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, -1)
    q = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, -1)
    n = 2 if mode == "chain" else 1 + m
    p = torch.rand(B, n, V, generator=g, device=DEV)
    p[:, 0] = row
    d = q.expand(B, n, V).reshape(B * n, V).contiguous()
    if mode == "best":
        tok = q.topk(m).indices.expand(B, m)
        d = None
    else:
        tok = torch.multinomial(q.expand(B, V), n - 1, replacement=True, generator=g)
    tok = torch.cat([torch.zeros_like(tok[:, :1]), tok], 1)
    par = torch.tensor([-1] + [0] * (n - 1), dtype=torch.int32, device=DEV).repeat(B)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    u = torch.rand(B * n, generator=g, device=DEV)
    count, path, token = tree.verify_tree(p.view(B * n, V), tok.reshape(-1), par, cu, n, uniforms=u,
                                          draft=d)
    first = torch.where(count > 1, tok.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
    freq = torch.bincount(first, minlength=V).double() / B
    sd = (row.double() * (1 - row.double()) / B).sqrt()
    assert bool(((freq - row.double()).abs() <= 5 * sd).all())
    rate = float((count > 1).double().mean())
    if mode == "chain":                   # accepted with probability sum min(p, q)
        want = float(torch.minimum(row, q).double().sum())
        assert abs(rate - want) <= 5 * math.sqrt(want * (1 - want) / B)
    assert 0 < rate < 1


def test_graph_and_streams():
    """Recorded calls of every mode replayed beside eager ones on another stream."""
    side = torch.cuda.Stream()
    for mode in ("chain", "drawn", "best", "greedy"):
        args = []
        for nodes, V in (([6, 9], 5000), ([30] * 5, 3001)):
            p, tokens, par, u, draft, _ = _case(nodes, V, mode, torch.float32, 6)
            cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
            args.append([None if x is None else x.to(DEV) for x in
                         (p, torch.tensor(tokens), torch.tensor(sum(par, []), dtype=torch.int32), cu,
                          u, draft)] + [max(nodes)])

        def call(a):
            return tree.verify_tree(*a[:4], a[6], uniforms=a[4], draft=a[5])
        want = [[x.clone() for x in call(a)] for a in args]
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(args[0])
        for _ in range(4):
            for x in out:
                x.fill_(-9)
            torch.cuda.synchronize()
            graph.replay()
            with torch.cuda.stream(side):
                got = call(args[1])
            torch.cuda.synchronize()
            for x, y in zip([*out, *got], [*want[0], *want[1]]):
                assert torch.equal(x, y), mode
