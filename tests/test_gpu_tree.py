"""Attention of trees of drafted tokens (tree.attn_tree) and their masks against 64-bit rows.

Tolerance: scores, softmax sums and outputs are held in 32 bits.  A score is a sum of 128
products in fp32; with inputs of about 0.7 its terms add up to 0.09 * 64 = 6 in absolute value, so
it is off by at most 128 * 2^-24 * 6 = 4.6e-5 and, roundings being of either sign, by 128^0.5 *
2^-24 * 6 = 4e-6 as a rule; a weight is off by that much of itself and the output by as much of the
largest |v|, to which a sum of n <= 2,500 weights adds n^0.5 2^-24 = 3e-6.  2e-5 of the largest |v|
is stated, and 2e-5 (5e-5 for the worst score above) for the log-sum-exp.  A bf16 output adds half
a step, 2^-8 of its value."""

import math

import pytest
import torch

from ananta_ocr_amd import ops, tree
from tree_oracle import ancestors, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 1.0 / math.sqrt(128)


def _trees(nodes, g, chain=False):
    out = []
    for n in nodes:
        out.append([-1][:n] + [i - 1 if chain else int(torch.randint(max(0, i - 6), i, (1,), generator=g))
                           for i in range(1, n)])
    return out


def _case(ctxs, nodes, H, Hkv, bs, lb, K, seed=0, page=None, paged=True, bad=True, chain=False):
    """A cache whose unseen slots (page ends, other sequences' nothing) hold NaN."""
    g = torch.Generator().manual_seed(seed)
    page = page or bs
    lens = [c + n for c, n in zip(ctxs, nodes)]
    P = max(1, max((n + page - 1) // page for n in lens))
    need = [(n + page - 1) // page for n in lens]
    pool = sum(need) + 2
    table = torch.full((len(lens), P), 10 ** 8, dtype=torch.int32)
    perm = torch.randperm(pool, generator=g)
    k = torch.randn(pool, page, Hkv, 128, generator=g) * 0.7
    v = torch.randn(pool, page, Hkv, 128, generator=g)
    o = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[o:o + need[b]].to(torch.int32)
        if bad and n % page:
            k[perm[o + need[b] - 1], n % page:] = math.nan
            v[perm[o + need[b] - 1], n % page:] = math.nan
        o += need[b]
    T = sum(nodes)
    q = (torch.randn(T, H, 128, generator=g) * 0.7).bfloat16()
    nblk = P * page // bs
    idx = torch.randint(-1, nblk + 2, (T, K), generator=g, dtype=torch.int32)
    bias = torch.randn(T, K, generator=g)
    valid = torch.rand(T, K, generator=g) < 0.8
    par = _trees(nodes, g, chain)
    k, v = k.bfloat16(), v.bfloat16()
    if not paged:
        k, v = (torch.stack([x[table[b].clamp(max=pool - 1).long()].reshape(P * page, Hkv, 128)
                             for b in range(len(lens))]).transpose(1, 2).contiguous() for x in (k, v))
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
    return dict(q=q, k=k, v=v, idx=idx, bias=bias, valid=valid, par=par, table=table, cu=cu,
                ctx=torch.tensor(ctxs, dtype=torch.int32), bs=bs, lw=lb * bs, page=page,
                paged=paged, nodes=nodes, ctxs=ctxs)


def _reference(c, seen=None):
    outs, lses = [], []
    for b, n in enumerate(c["nodes"]):
        r0, S = int(c["cu"][b]), c["ctxs"][b] + n
        if c["paged"]:
            t = c["table"][b, :(S + c["page"] - 1) // c["page"]].long()
            k, v = (c[x][t].reshape(-1, *c[x].shape[2:])[:S] for x in "kv")
        else:
            k, v = (c[x][b, :, :S].transpose(0, 1) for x in "kv")
        chains = [ancestors(c["par"][b], i) for i in range(n)]
        rows = slice(r0, r0 + n)
        o, l = attend(c["q"][rows], k, v, c["idx"][rows], c["bias"][rows], c["valid"][rows],
                      chains if seen is None else [seen(b, i) for i in range(n)],
                      [len(x) - 1 for x in chains], c["ctxs"][b], c["bs"], c["lw"], SCALE)
        outs.append(o)
        lses.append(l)
    return torch.cat(outs), torch.cat(lses)


def _run(c, mask=None, **kw):
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "idx", "bias", "valid", "table", "ctx", "cu")}
    par = torch.tensor(sum(c["par"], []), dtype=torch.int32, device=DEV)
    n = max(c["nodes"])
    m, depth = tree.tree_masks(par, d["cu"], n)
    paging = dict(block_table=d["table"], page_size=c["page"]) if c["paged"] else {}
    return tree.attn_tree(d["q"], d["k"], d["v"], d["idx"], d["bias"], d["valid"],
                          m if mask is None else mask.to(DEV), depth, d["ctx"], d["cu"], n,
                          c["bs"], c["lw"], SCALE, **paging, **kw)


def _close(out, lse, ref, ref_lse, v_max, what=""):
    out, lse = out.cpu(), lse.cpu()
    tol = 2e-5 * v_max + (2.0 ** -8 * ref.abs() if out.dtype == torch.bfloat16 else 0.0)
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what} {err.max().item()}"
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert not out[none].any()
    assert float((lse.double() - ref_lse)[~none].abs().max() if (~none).any() else 0.0) <= 5e-5, what


CASES = [
    # contexts, nodes, H, Hkv, bs, lb, K
    ([300], [8], 2, 2, 64, 2, 4),
    ([0, 1, 700, 129], [5, 1, 17, 3], 2, 2, 64, 2, 8),      # no context, one token
    ([333, 1000], [13, 32], 10, 2, 32, 4, 12),              # shared key heads
    ([640, 64], [33, 64], 4, 1, 64, 1, 3),                  # one key head, whole blocks
    ([500, 80], [65, 100], 2, 2, 32, 4, 16),                # two mask words
    ([900], [256], 2, 1, 64, 8, 16),                        # the largest tree
    ([1500, 40], [7, 0], 2, 2, 64, 2, 33),                  # a request without nodes, many slots
    ([2000], [3], 2, 2, 64, 30, 64),
]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_rows_match_64_bits(case, paged):
    c = _case(*case, paged=paged)
    out, lse = _run(c, return_lse=True)
    ref, ref_lse = _reference(c)
    _close(out, lse, ref, ref_lse, 5.0, str(case))
    b16, _ = _run(c, return_lse=True, out_dtype=torch.bfloat16)
    _close(b16, lse, ref, ref_lse, 5.0, str(case))


@pytest.mark.parametrize("case", [
    ([5000], [32], 2, 2, 32, 2, 64), ([5000, 900], [64, 33], 2, 2, 32, 2, 64),
    ([5000], [128], 2, 1, 32, 2, 64), ([64 * 90], [50], 4, 2, 64, 1, 64)])
def test_the_most_slots(case):
    """64 slots a row in every height of the row tiles: the largest tables of slots beside the stages."""
    c = _case(*case)
    out, lse = _run(c, return_lse=True)
    _close(out, lse, *_reference(c), 5.0, str(case))


@pytest.mark.parametrize("bs,page", [(64, 128), (32, 96), (128, 128), (32, 64)])
def test_pages_of_several_blocks(bs, page):
    c = _case([777, 130], [9, 20], 4, 2, bs, 2, 6, page=page)
    out, lse = _run(c, return_lse=True)
    _close(out, lse, *_reference(c), 5.0)


def test_masks_and_depths():
    g = torch.Generator().manual_seed(3)
    nodes = [1, 0, 256, 70, 64]
    par = _trees(nodes, g)
    par[3][5] = 40                        # not an earlier node: none
    par[3][6] = -7
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32).to(DEV)
    mask, depth = tree.tree_masks(torch.tensor(sum(par, [])).to(DEV), cu, 256)
    mask, depth, r = mask.cpu(), depth.cpu().tolist(), 0
    for p in par:
        for i in range(len(p)):
            a = ancestors(p, i)
            got = [m for m in range(256) if (int(mask[r, m // 64]) >> (m % 64)) & 1]
            assert got == sorted(a) and depth[r] == len(a) - 1
            r += 1


def test_masks_of_the_callers_own_and_rows_that_see_nothing():
    """Any set of drafted nodes, the row itself not among them; without context such a row is
    empty, and the other rows stay as they are."""
    c = _case([0, 200], [6, 6], 2, 2, 64, 1, 2, seed=4)
    rows = {(0, 0): [], (0, 1): [3, 5], (0, 2): [], (0, 3): [0], (0, 4): [1], (0, 5): [5],
            (1, 0): [], (1, 1): [0, 1], (1, 2): [5], (1, 3): [3], (1, 4): [], (1, 5): [2]}
    mask = torch.tensor([[sum(1 << m for m in rows[b, i])] for b in range(2) for i in range(6)])
    out, lse = _run(c, mask=mask, return_lse=True)
    _close(out, lse, *_reference(c, lambda b, i: rows[b, i]), 5.0)
    assert (lse[0] == -math.inf).all() and not out[0].any()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Hkv,bs,lb", [(2, 64, 2), (1, 32, 3)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(value, Hkv, bs, lb):
    """V and K of a drafted node, of a key below the windows that few rows name and of a window key
    of the first rows only."""
    c = _case([600], [20], 2, Hkv, bs, lb, 4, seed=9)
    blk = 1
    c["idx"][:, 0] = -1
    c["idx"][3, 0], c["valid"][3, 0] = blk, True
    c["idx"][:, 1:] = torch.where(c["idx"][:, 1:] == blk, -1, c["idx"][:, 1:])

    def slot(j):
        return int(c["table"][0, j // c["page"]]), j % c["page"]
    first = 600 - c["lw"] + 1             # the window's first key at depth 0
    for x, j in (("v", 600 + 7), ("v", blk * bs + 3), ("v", first), ("k", 600 + 11)):
        c[x][slot(j)] = value
    out, lse = _run(c, return_lse=True)
    ref, ref_lse = _reference(c)
    out, lse = out.cpu().double(), lse.cpu().double()
    fine = ref.isfinite().all(-1).all(-1) & ~ref_lse.isnan().any(-1)
    assert 0 < int(fine.sum()) < 20
    assert float((out - ref)[fine].abs().max()) <= 1e-4
    assert not out[~fine].isfinite().all()
    hit = [i for i in range(20) if 7 in ancestors(c["par"][0], i)]
    clean = [i for i in range(20) if bool(fine[i])]
    assert hit and not set(hit) & set(clean)
    # the very values, where only V is not finite
    only_v = [i for i in range(20) if not bool(fine[i]) and 11 not in ancestors(c["par"][0], i)]
    same = out[only_v].nan_to_num(5.0, 6.0, 7.0) - ref[only_v].nan_to_num(5.0, 6.0, 7.0)
    assert float(same.abs().max()) <= 1e-4


def test_repeated_invalid_and_outside_slots():
    c = _case([1000], [4], 2, 2, 64, 2, 8, seed=5)
    c["idx"][:] = torch.tensor([3, 3, 20, 3, 10 ** 9, -5, 14, 5], dtype=torch.int32)
    c["valid"][:] = torch.tensor([0, 1, 1, 1, 1, 1, 1, 1], dtype=torch.bool)
    out, lse = _run(c, return_lse=True)
    _close(out, lse, *_reference(c), 5.0)


def test_no_routed_blocks_is_dense_attention_over_a_long_window():
    c = _case([450, 77], [12, 30], 4, 2, 64, 16, 1, seed=6)
    c["idx"][:] = -1
    ref, ref_lse = _reference(c)
    out, lse = _run(c, return_lse=True)
    _close(out, lse, ref, ref_lse, 5.0)
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "table", "ctx", "cu")}
    par = torch.tensor(sum(c["par"], []), dtype=torch.int64, device=DEV)
    m, depth = tree.tree_masks(par, d["cu"], 30)
    out, lse = tree.attn_tree(d["q"], d["k"], d["v"], None, None, None, m, depth, d["ctx"].long(),
                              d["cu"].long(), 30, 64, 1024, SCALE, block_table=d["table"].long(),
                              page_size=64, return_lse=True)
    _close(out, lse, ref, ref_lse, 5.0)


def test_strides_of_queries_and_caches():
    """Queries out of a wider projection, keys and values of one interleaved pool, a contiguous
    cache stored [B, S, H, D]."""
    c = _case([400, 90], [9, 11], 4, 2, 64, 2, 4, seed=7)
    ref = _reference(c)
    pool = torch.stack([c["k"], c["v"]], 1).to(DEV)           # [pages, 2, page, Hkv, D]
    wide = torch.randn(c["q"].shape[0], 3, 4, 128).bfloat16().to(DEV)
    wide[:, 1] = c["q"].to(DEV)
    d = {x: c[x].to(DEV) for x in ("idx", "bias", "valid", "table", "ctx", "cu")}
    par = torch.tensor(sum(c["par"], []), dtype=torch.int32, device=DEV)
    m, depth = tree.tree_masks(par, d["cu"], 11)
    for q in (wide[:, 1], c["q"].to(DEV).transpose(1, 2).contiguous().transpose(1, 2)):
        out, lse = tree.attn_tree(q, pool[:, 0], pool[:, 1], d["idx"], d["bias"], d["valid"], m, depth,
                                  d["ctx"], d["cu"], 11, 64, 128, SCALE, block_table=d["table"],
                                  page_size=64, return_lse=True)
        _close(out, lse, *ref, 5.0)
    f = _case([400, 90], [9, 11], 4, 2, 64, 2, 4, seed=7, paged=False)
    ref = _reference(f)
    f["k"], f["v"] = (f[x].transpose(1, 2).contiguous().transpose(1, 2) for x in "kv")
    _close(*_run(f, return_lse=True), *ref, 5.0)


def test_cache_past_32_bit_offsets():
    """Pages at the far end of a pool of more than 2^32 bytes and 2^31 elements."""
    c = _case([300], [9], 10, 10, 64, 2, 4, seed=8)
    far = 27000                           # pages: 27,000 x 64 x 10 x 128 = 2.2e9 elements
    used = c["table"][0].long()
    big = {}
    for x in "kv":
        t = torch.empty(far, 64, 10, 128, dtype=torch.bfloat16, device=DEV)
        t[far - used.numel():] = c[x][used].to(DEV)
        big[x] = t
    ref = _reference(c)
    d = {x: c[x].to(DEV) for x in ("q", "idx", "bias", "valid", "ctx", "cu")}
    table = torch.arange(far - used.numel(), far, dtype=torch.int32, device=DEV)[None]
    m, depth = tree.tree_masks(torch.tensor(c["par"][0], device=DEV), d["cu"], 9)
    out, lse = tree.attn_tree(d["q"], big["k"], big["v"], d["idx"], d["bias"], d["valid"], m, depth,
                              d["ctx"], d["cu"], 9, 64, 128, SCALE, block_table=table, page_size=64,
                              return_lse=True)
    _close(out, lse, *ref, 5.0)


def test_chain_equals_the_extend_rows():
    """A tree without branches is a chunk of known tokens: ops.attn_extend's rows."""
    c = _case([640, 200], [20, 33], 2, 2, 64, 4, 8, seed=11, chain=True, bad=False)
    out = _run(c)
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "idx", "bias", "valid", "table", "ctx", "cu")}
    d["table"] = d["table"].clamp(max=c["k"].shape[0] - 1)
    ref = ops.attn_extend(d["q"], d["k"], d["v"], d["idx"], d["bias"], d["valid"],
                          d["ctx"] + torch.tensor(c["nodes"], device=DEV), d["ctx"], d["cu"], 33,
                          d["table"], 64, 256, SCALE)
    assert float((out - ref).abs().max()) <= 4e-5


def test_rows_do_not_depend_on_the_other_requests():
    """The batch, and each request alone: the same to the order of the sums."""
    c = _case([640, 200, 1500], [20, 33, 7], 4, 2, 64, 4, 8, seed=12)
    whole = _run(c).cpu()
    for b in range(3):
        r0, r1 = int(c["cu"][b]), int(c["cu"][b + 1])
        one = dict(c, nodes=[c["nodes"][b]], ctxs=[c["ctxs"][b]], par=[c["par"][b]],
                   table=c["table"][b:b + 1], ctx=c["ctx"][b:b + 1], cu=c["cu"][b:b + 2] - r0,
                   **{x: c[x][r0:r1] for x in ("q", "idx", "bias", "valid")})
        alone = _run(one).cpu()
        assert float((alone - whole[r0:r1]).abs().max()) <= 2e-5 * 5


def test_graph_streams_and_repeats():
    """A recorded call replayed between eager ones of another shape on another stream, its inputs
    rewritten before each replay: the eager bits every time."""
    c, e = (_case([500, 90], [9, 11], 4, 2, 64, 2, 4, seed=s) for s in (1, 2))
    other = _case([2000, 300, 40], [30, 12, 3], 4, 2, 64, 4, 8, seed=3)
    want = [_run(x).clone() for x in (c, e, other)]
    for x in (c, e, other):
        x["par_d"] = torch.tensor(sum(x["par"], []), dtype=torch.int32, device=DEV)
        for y in ("q", "k", "v", "idx", "bias", "valid", "table", "ctx", "cu"):
            x[y + "_d"] = x[y].to(DEV)

    def call(x):
        m, depth = tree.tree_masks(x["par_d"], x["cu_d"], max(x["nodes"]))
        return tree.attn_tree(x["q_d"], x["k_d"], x["v_d"], x["idx_d"], x["bias_d"], x["valid_d"], m,
                              depth, x["ctx_d"], x["cu_d"], max(x["nodes"]), 64, x["lw"], SCALE,
                              block_table=x["table_d"], page_size=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(c)
    names = [y + "_d" for y in ("q", "k", "v", "idx", "bias", "valid", "table", "par")]
    first = {y: c[y].clone() for y in names}
    for i in range(4):
        for y in names:
            c[y].copy_((e if i % 2 else first)[y])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            got = call(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2]) and torch.equal(got, want[2])


def test_batches_padded_to_a_fixed_size():
    """Rows past the last tree, and prefix sums past the rows: the trees' rows as without them."""
    c = _case([300, 65], [9, 6], 4, 2, 64, 2, 4, seed=13)
    ref = _reference(c)
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "idx", "bias", "valid", "table", "ctx", "cu")}
    par = torch.tensor(sum(c["par"], []), dtype=torch.int32, device=DEV)
    pad = {x: torch.cat([d[x], torch.ones_like(d[x][:7])]) for x in ("q", "idx", "bias", "valid")}
    par_p = torch.cat([par, torch.full_like(par[:7], 3)])
    table = torch.cat([d["table"], torch.full_like(d["table"], -5)])
    ctx = torch.cat([d["ctx"], torch.tensor([10 ** 6, -7], dtype=torch.int32, device=DEV)])
    cu = torch.cat([d["cu"], torch.tensor([15, 15], dtype=torch.int32, device=DEV)])
    mask, depth = tree.tree_masks(par_p, cu, 32)
    out, lse = tree.attn_tree(pad["q"], d["k"], d["v"], pad["idx"], pad["bias"], pad["valid"], mask, depth,
                              ctx, cu, 32, 64, 128, SCALE, block_table=table, page_size=64,
                              return_lse=True)
    assert out.shape[0] == 22
    _close(out[:15], lse[:15], *ref, 5.0)
    # a third and a fourth request that claim rows there are not
    cu[3:] = torch.tensor([10 ** 6], device=DEV)
    mask, depth = tree.tree_masks(par_p[:15], cu, 32)
    out, lse = tree.attn_tree(d["q"], d["k"], d["v"], d["idx"], d["bias"], d["valid"], mask, depth, ctx, cu,
                              32, 64, 1 << 40, SCALE, block_table=table, page_size=64, return_lse=True)
    wide = dict(c, lw=1 << 20)
    _close(out, lse, *_reference(wide), 5.0)


def test_contexts_past_the_cache_are_cut_to_it():
    """More context than the table holds: its last keys, and no drafted ones."""
    c = _case([128], [4], 2, 2, 64, 8, 2, seed=14, bad=False)
    c["idx"][:] = -1
    long = dict(c, ctx=torch.tensor([5000], dtype=torch.int32))
    out = _run(long)
    d = c["table"][0, :3].long()
    k, v = (c[x][d].reshape(-1, 2, 128) for x in "kv")
    depth = [len(ancestors(c["par"][0], i)) - 1 for i in range(4)]
    ref, _ = attend(c["q"], k, v, None, None, None, [[]] * 4, depth, 192, 64, 512, SCALE)
    assert float((out.cpu().double() - ref).abs().max()) <= 1e-4
