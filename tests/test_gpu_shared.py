"""Attention of batches that share prompts (shared_prefix.attn_shared) against 64-bit rows.

Tolerance: as for the attention of trees.  Scores, sums and outputs are held in 32 bits: a score is a sum
of 128 products of inputs of about 0.7, whose absolute values add up to 6, so it is off by at most 128 *
2^-24 * 6 = 4.6e-5 and, roundings being of either sign, by 128^0.5 * 2^-24 * 6 = 4e-6 as a rule; a weight
is off by that much of itself and the output by as much of the largest |v|; a sum of n weights adds n^0.5 *
2^-24, 7e-6 for 14,000.  3e-5 of the largest |v| is stated, and 5e-5 for the log-sum-exp.  A bf16 output
adds half a step, 2^-8 of its value."""

import math

import pytest
import torch

from ananta_ocr_amd import shared_prefix

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 1.0 / math.sqrt(128)
I32 = torch.int32


def _case(groups, H, Hkv, page, seed=0, spare_rows=0, alone=()):
    """groups: (prefix, [(context, new), ...]) each; alone: sequences of no group, behind them.  Pages at
    random, a group's whole pages of the prefix in common; unwritten slots hold NaN, entries past a
    sequence numbers that name no page."""
    g = torch.Generator().manual_seed(seed)
    seqs = [(p, i, c, n) for i, (p, some) in enumerate(groups) for c, n in some]
    seqs += [(0, -1, c, n) for c, n in alone]
    lens = [c + n for _, _, c, n in seqs]
    need = [(n + page - 1) // page for n in lens]
    P = max(need + [1]) + 1
    pool = sum(need) + 3
    free = torch.randperm(pool, generator=g).tolist()
    k = torch.full((pool, page, Hkv, 128), math.nan)
    v = torch.full((pool, page, Hkv, 128), math.nan)
    table = torch.full((len(seqs), P), 10 ** 8, dtype=I32)
    firsts, keys = {}, []
    for b, (p, i, c, n) in enumerate(seqs):
        S = c + n
        kb, vb = torch.randn(S, Hkv, 128, generator=g) * 0.7, torch.randn(S, Hkv, 128, generator=g)
        mine = [free.pop() for _ in range(need[b])]
        if i in firsts:                       # the prompt's keys, and whole pages of it
            row, k0, v0 = firsts[i]
            m = min(p, S, len(k0))
            kb[:m], vb[:m] = k0[:m], v0[:m]
            mine[:m // page] = row[:m // page]
        elif i >= 0:
            firsts[i] = mine, kb, vb
        kb, vb = kb.bfloat16(), vb.bfloat16()
        for j, pg in enumerate(mine):
            some = slice(j * page, min((j + 1) * page, S))
            k[pg, :some.stop - some.start], v[pg, :some.stop - some.start] = kb[some].float(), vb[some].float()
        table[b, :need[b]] = torch.tensor(mine, dtype=I32)
        keys.append((kb, vb))
    new = [n for _, _, _, n in seqs]
    T = sum(new)
    q = (torch.randn(T + spare_rows, H, 128, generator=g) * 0.7).bfloat16()
    ways = [len(some) for _, some in groups]

    def sums(x):
        return torch.tensor([0] + x, dtype=torch.int64).cumsum(0).to(I32)

    return dict(q=q, k=k.bfloat16(), v=v.bfloat16(), table=table, ctx=torch.tensor([c for _, _, c, _ in seqs],
                                                                                 dtype=I32),
                cu=sums(new), groups=sums(ways), prefix=torch.tensor([p for p, _ in groups], dtype=I32),
                keys=keys, new=new, T=T)


def _reference(c):
    H, Hkv = c["q"].shape[1], c["k"].shape[2]
    outs, lses, r = [], [], 0
    for (k, v), n, ctx in zip(c["keys"], c["new"], c["ctx"].tolist()):
        if n == 0:
            continue
        k, v = (x.to(DEV).double().repeat_interleave(H // Hkv, 1).transpose(0, 1).contiguous() for x in (k, v))
        z = torch.matmul(c["q"][r:r + n].to(DEV).double().transpose(0, 1), k.transpose(1, 2).contiguous()) * SCALE
        j, t = torch.arange(k.shape[1], device=DEV), ctx + torch.arange(n, device=DEV)
        z = torch.where(j <= t[:, None], z, -math.inf)
        lses.append(torch.logsumexp(z, -1).t())
        outs.append(torch.matmul(torch.softmax(z, -1), v).transpose(0, 1))
        r += n
    return torch.cat(outs), torch.cat(lses)


def _run(c, groups=True, **kw):
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "table", "ctx", "cu", "groups", "prefix")}
    return shared_prefix.attn_shared(d["q"], d["k"], d["v"], d["table"], d["ctx"], d["cu"],
                                     d["groups"] if groups else None, d["prefix"] if groups else None, SCALE, **kw)


def _check(c, out, lse, v_max=None):
    ref, ref_lse = _reference(c)
    T = c["T"]
    v_max = max(float(v.float().abs().max()) for _, v in c["keys"] if v.numel()) if v_max is None else v_max
    tol = 3e-5 * v_max + (2.0 ** -8 * ref.abs() if out.dtype == torch.bfloat16 else 0.0)
    err = (out[:T].double() - ref).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()
    assert float((lse[:T].double() - ref_lse).abs().max()) <= 5e-5
    assert not out[T:].any() and bool((lse[T:] == -math.inf).all())


CASES = [
    # groups (prefix, [(context, new)]), H, Hkv, page, sequences of no group
    ([(0, [(0, 1)])], 1, 1, 64, ()),                                     # one token
    ([(128, [(128, 1), (130, 1), (200, 1)])], 2, 2, 64, ()),
    ([(100, [(100, 1), (100, 1)]), (65, [(80, 1)])], 2, 2, 64, ()),      # prompts that end inside a page
    ([(640, [(641 + 13 * i, 1) for i in range(33)])], 2, 1, 64, ()),     # more than 32 rows
    ([(300, [(301 + i, 1) for i in range(13)]), (17, [(40, 1)])], 10, 2, 16, ()),
    ([(100, [(100, 5), (103, 1), (190, 17)])], 4, 2, 32, ()),            # several rows a sequence
    ([(1000, [(1000, 70), (1200, 3)])], 10, 1, 64, ()),                  # tiles of rows
    ([(0, [(0, 33)]), (0, [(5, 7), (0, 1)])], 2, 2, 64, ()),             # nothing shared
    ([(50, [(50, 0), (60, 2), (55, 0)])], 2, 2, 64, ()),                 # sequences without rows
    ([(5, [(6, 1), (9, 2)]), (40, [(41, 1)])], 3, 3, 1, ((7, 1), (0, 3))),       # pages of a token
    ([(90, [(95, 2), (99, 1)])], 2, 2, 7, ((3, 1),)),
    ([], 2, 2, 64, ((100, 1), (5, 3), (0, 1), (700, 1))),                # no group
    ([(64, [(64 + i, 1) for i in range(300)])], 1, 1, 64, ()),           # many sequences
    ([(10, [(12, 1)])] * 90, 1, 1, 16, ((5, 1),) * 70),                  # many groups
    ([(7000, [(7000, 1), (7001, 4), (9000, 2)])], 2, 2, 64, ()),
    ([(500, [(500 + 7 * i, 129) for i in range(3)])], 2, 1, 128, ()),
]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_64_bits(case, out):
    groups, H, Hkv, page, alone = CASES[case]
    c = _case(groups, H, Hkv, page, case, spare_rows=case % 3, alone=alone)
    _check(c, *_run(c, out_dtype=out, return_lse=True))


def test_bf16_is_the_fp32_output_rounded_once():
    c = _case([(900, [(901 + i, 1) for i in range(20)])], 4, 2, 64, 5)
    assert torch.equal(_run(c, out_dtype=torch.bfloat16), _run(c).bfloat16())


@pytest.mark.parametrize("case", [1, 4, 6])
def test_sharing_changes_nothing_but_rounding(case):
    groups, H, Hkv, page, alone = CASES[case]
    c = _case(groups, H, Hkv, page, 31, alone=alone)
    _check(c, *_run(c, return_lse=True))
    _check(c, *_run(c, groups=False, return_lse=True))


def test_prompts_past_the_positions_of_some_rows():
    """A prefix longer than some of its sequences: their rows see the keys up to themselves."""
    c = _case([(500, [(600, 1), (20, 3), (499, 2), (0, 1)])], 2, 2, 64, 9)
    c["prefix"][0] = 10 ** 9
    _run(c)                                      # (read through the first row: in bounds)
    c["prefix"][0] = 500
    k0, v0 = c["keys"][0]
    for b in (1, 2, 3):
        n = len(c["keys"][b][0])
        m = min(n, 500)
        assert torch.equal(c["keys"][b][0][:m], k0[:m])
    _check(c, *_run(c, return_lse=True))


def test_values_that_are_not_finite():
    """Keys and values that a row does not see leave it alone, those that it sees do not: later tokens of
    its sequence, other sequences', and the prompt's."""
    c = _case([(128, [(130, 4), (140, 3)])], 2, 2, 64, 12)
    clean, clean_lse = _run(c, return_lse=True)
    t, page = c["table"], 64

    def slot(b, j):
        return int(t[b, j // page]), j % page

    for value in (math.nan, math.inf, -math.inf):
        d = dict(c, k=c["k"].clone(), v=c["v"].clone())
        d["v"][slot(0, 132)][1, 7] = value               # head 1's key of row 2 of sequence 0
        out, lse = _run(d, return_lse=True)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[2:4, 1, 7] = True                            # rows 2 and 3 see it
        assert torch.equal(~torch.isfinite(out), bad)
        assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse, clean_lse)
        d = dict(c, k=c["k"].clone(), v=c["v"].clone())
        d["k"][slot(1, 142)][0, 3] = math.nan            # a key of sequence 1's last row
        out, _ = _run(d, return_lse=True)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[6, 0] = True
        assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])
        d = dict(c, k=c["k"].clone(), v=c["v"].clone())
        d["v"][slot(0, 100)][0, 5] = value               # the prompt's: every row
        out, _ = _run(d, return_lse=True)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[:, 0, 5] = True
        assert torch.equal(~torch.isfinite(out), bad) and torch.equal(out[~bad], clean[~bad])


def test_strides_and_layers():
    """Caches and queries as views: a layer of a pool, keys beside values, queries of a projection."""
    c = _case([(128, [(130, 1), (200, 2)])], 4, 2, 32, 14)
    want = _run(c)
    pool, page = c["k"].shape[:2]
    both = torch.randn(pool, 3, page, 2, 2, 128).bfloat16().to(DEV)
    both[:, 1, :, 0], both[:, 1, :, 1] = c["k"].to(DEV), c["v"].to(DEV)
    qkv = torch.randn(c["q"].shape[0], 8, 128).bfloat16().to(DEV)
    qkv[:, 2:6] = c["q"].to(DEV)
    out = shared_prefix.attn_shared(qkv[:, 2:6], both[:, 1, :, 0], both[:, 1, :, 1], c["table"].to(DEV).long(),
                                    c["ctx"].to(DEV).long(), c["cu"].to(DEV).long(), c["groups"].to(DEV),
                                    c["prefix"].to(DEV), SCALE)
    assert torch.equal(out, want)


def test_sums_that_do_not_fit():
    """Prefix sums past the rows and the batch, or that fall, touch nothing else; lengths outside the
    table are cut to it."""
    c = _case([(64, [(64 + i, 1) for i in range(6)])], 2, 2, 64, 15)
    for cu, gr, pre, ctx in (([0, 1, 2, 3, 900, 901, 10 ** 9], [0, 10 ** 6], [64], None),
                             ([0, 6, 0, 6, 0, 6, 6], [0, 6], [64], None), ([6, 5, 4, 3, 2, 1, 0], [6, 0], [64], None),
                             ([-5, 1, 2, 3, 4, 5, 6], [-7, 6], [-3], None),
                             ([0, 1, 2, 3, 4, 5, 6], [0, 6, 0, 6, 0, 6], [64] * 5, [-9, 10 ** 9, 0, 5, 7, 2 ** 31 - 1])):
        d = dict(c, cu=torch.tensor(cu, dtype=I32), groups=torch.tensor(gr, dtype=I32),
                 prefix=torch.tensor(pre, dtype=I32))
        if ctx:
            d["ctx"] = torch.tensor(ctx, dtype=I32)
        assert _run(d).shape == (6, 2, 128)
    torch.cuda.synchronize()
    _check(c, *_run(c, return_lse=True))


def test_empty_batches():
    q = torch.zeros(3, 2, 128, device=DEV).bfloat16()
    k = torch.zeros(4, 16, 2, 128, device=DEV).bfloat16()
    i = torch.zeros(0, dtype=I32, device=DEV)
    one = torch.zeros(1, dtype=I32, device=DEV)
    out, lse = shared_prefix.attn_shared(q, k, k, i.view(0, 5), i, one, one, i, SCALE, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    out = shared_prefix.attn_shared(q[:0], k, k, one.view(1, 1), one, torch.zeros(2, dtype=I32, device=DEV), None,
                                    None, SCALE)
    assert out.shape == (0, 2, 128)
    for kk, table in ((k[:0], one.view(1, 1)), (k, one.view(1, 1)[:, :0])):        # no pages, no entries
        out, lse = shared_prefix.attn_shared(q, kk, kk, table, one, torch.tensor([0, 3], dtype=I32, device=DEV),
                                             None, None, SCALE, return_lse=True)
        assert not out.any() and bool((lse == -math.inf).all())


def test_in_a_graph_with_other_lengths():
    """Captured once; replays with other lengths, groups and tables against eager calls."""
    cases = [_case([(640, [(641 + 9 * i, 1) for i in range(5)]), (64, [(70, 1)] * 3)], 4, 2, 64, 16),
             _case([(64, [(70, 1)] * 2), (300, [(900, 1)] * 6)], 4, 2, 64, 17),
             _case([(0, [(0, 1)]), (10, [(10, 1)] * 7)], 4, 2, 64, 18)]
    P, pool = max(c["table"].shape[1] for c in cases), max(c["k"].shape[0] for c in cases)
    buf = {}
    for c in cases:
        c["table"] = torch.nn.functional.pad(c["table"], (0, P - c["table"].shape[1]), value=-1)
        for x in "kv":
            c[x] = torch.cat([c[x], c[x][:1].expand(pool - len(c[x]), -1, -1, -1)])
    names = ("q", "k", "v", "table", "ctx", "cu", "groups", "prefix")
    buf = {x: cases[0][x].to(DEV) for x in names}
    args = buf["q"], buf["k"], buf["v"], buf["table"], buf["ctx"], buf["cu"], buf["groups"], buf["prefix"], SCALE
    shared_prefix.attn_shared(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = shared_prefix.attn_shared(*args, return_lse=True)
    for c in cases + cases[:1]:
        for x in names:
            buf[x].copy_(c[x])
        graph.replay()
        torch.cuda.synchronize()
        _check(c, out, lse)
        want, want_lse = shared_prefix.attn_shared(*args, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_two_streams_at_once():
    a = _case([(2000, [(2001 + i, 1) for i in range(8)])], 10, 10, 64, 20)
    b = _case([(900, [(901 + i, 2) for i in range(5)])], 10, 10, 64, 21)
    want = _run(a), _run(b)
    da, db = ({x: c[x].to(DEV) for x in ("q", "k", "v", "table", "ctx", "cu", "groups", "prefix")} for c in (a, b))
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(4):
        for i, d in enumerate((da, db)):
            with torch.cuda.stream(streams[i]):
                got[i].append(shared_prefix.attn_shared(*(d[x] for x in ("q", "k", "v", "table", "ctx", "cu",
                                                                         "groups", "prefix")), SCALE))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_past_32_bits():
    """Pages whose bytes lie past 2^32 (elements past 2^31) of a cache."""
    pages = 2 ** 31 // (64 * 2 * 128) + 70
    k = torch.zeros(pages, 64, 2, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(pages, 64, 2, 128, dtype=torch.bfloat16, device=DEV)
    c = _case([(128, [(130, 1), (200, 2)])], 4, 2, 64, 22)
    n = len(c["k"])
    k[-n:], v[-n:] = c["k"].to(DEV), c["v"].to(DEV)
    d = dict(c, table=torch.where(c["table"] < n, c["table"] + (pages - n), c["table"]), k=k, v=v)
    assert torch.equal(_run(d), _run(c))


def _padded(c, n):
    """The same with n more sequences, without rows."""
    more = dict(c)
    more["table"] = torch.cat([c["table"], c["table"][:1].expand(n, -1)])
    more["ctx"] = torch.cat([c["ctx"], torch.full((n,), 9, dtype=I32)])
    more["cu"] = torch.cat([c["cu"], c["cu"][-1:].expand(n)])
    return more


@pytest.mark.parametrize("case", [1, 4, 5, 6, 8, 9, 14, 15])
def test_more_sequences_than_a_wavefront_changes_nothing(case):
    """A batch of up to 64 sequences plans its work inside of the attention, a larger one before it: the same units,
    the same sums."""
    groups, H, Hkv, page, alone = CASES[case]
    c = _case(groups, H, Hkv, page, case, spare_rows=2, alone=alone)
    B = len(c["ctx"])
    out, lse = _run(c, return_lse=True)
    _check(c, out, lse)
    for n in (64 - B, 65 - B, 300):
        o, l = _run(_padded(c, n), return_lse=True)
        assert torch.equal(o, out) and torch.equal(l, lse), n


def test_64_groups():
    for n in (64, 65):
        c = _case([(10 + i, [(12 + i, 1 + i % 2)]) for i in range(n)], 1, 1, 16, 3)
        _check(c, *_run(c, return_lse=True))


@pytest.mark.parametrize("B, n, ctx", [(40, 1, 4000), (1, 1000, 9000), (3, 60, 48000)])
def test_more_units_than_a_pass(B, n, ctx):
    """More than 64 units a work-group, at one, four and two row tiles: 32 key heads, whose sequences' tables name the
    same pages."""
    g = torch.Generator().manual_seed(B)
    H, page = 32, 64
    pages = 150
    k, v = ((torch.randn(pages, page, H, 128, generator=g) * 0.7).bfloat16() for _ in range(2))
    P = (ctx + n + page - 1) // page
    c = dict(q=(torch.randn(B * n, H, 128, generator=g) * 0.7).bfloat16(), k=k, v=v,
             table=torch.stack([torch.randint(0, pages, (P,), generator=g) for _ in range(B)]).to(I32),
             ctx=torch.full((B,), ctx, dtype=I32), cu=torch.arange(B + 1, dtype=I32) * n, T=B * n,
             groups=torch.tensor([0, 1], dtype=I32), prefix=torch.zeros(1, dtype=I32), new=[n] * B)
    out, lse = _run(c, groups=False, return_lse=True)
    more = _padded(c, 70)
    # (an average of rows that keeps the row tile: padded by a group, of one sequence without a prompt)
    o, l = _run(more, groups=B == 1, return_lse=True)
    c["keys"] = [tuple(x[t.long()].reshape(-1, H, 128)[:ctx + n] for x in (k, v)) for t in c["table"][:1]]
    first = {**c, "new": [n], "ctx": c["ctx"][:1], "T": n, "q": c["q"][:n]}
    _check(first, out[:n], lse[:n])
    tol = 6e-5 * float(v.float().abs().max())
    assert float((o - out).abs().max()) <= tol and float((l - lse).abs().max()) <= 1e-4
