"""Measured cases of the speculative decoding operators over a paged cache: a tree of drafted
tokens attends its sequence's cache (``tree``), the target's probabilities decide which of the
drafted tokens stand (``verify``), and the pages of the cache are kept in order around it:
accepted rows moved up (``keep``), sequences forked, grown and freed (``fork``), the pool
compacted (``compact``).

A tree is packed: rows cu[b] .. cu[b + 1] - 1 are the nodes of sequence b, node 0 its root (the
newest sampled token), every other node's parent an earlier node.  Node i's key and value lie in
the cache at slot context_len + i, its position is context_len + depth.

Heads (10), head and index dim (128), blocks of 32 with 4 local and 12 routed blocks and blocks
of 64 with windows of 512 and 1,024 and 8 or 16 routed blocks are those of the checkpoint's
configuration and of the benchmark; sequences hold 10 to 100 pages of 273 tokens.  Vocabularies
are generic.
"""

import math
import random
from types import SimpleNamespace

import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------ the cases

def listed():
    return [
        # One request with a small draft on a ten-page prompt: latency and launches.
        dict(name="tree_b1_n8", kind="tree", B=1, n_lo=8, n_hi=8, lo=2730, hi=2730, bs=64, lb=8,
             K=8, H=10, Hkv=10, paged=True, out="fp32", layout=0),
        # Few requests of a long-document batch, trees of ordinary size.
        dict(name="tree_b8_n32", kind="tree", B=8, n_lo=16, n_hi=32, lo=27300, hi=27300, bs=64,
             lb=16, K=16, H=10, Hkv=10, paged=True, out="bf16", layout=1),
        # A full serving batch of 10 to 100 pages with wide trees.
        dict(name="tree_b32_n64", kind="tree", B=32, n_lo=24, n_hi=64, lo=2730, hi=27300, bs=64,
             lb=16, K=16, H=10, Hkv=10, paged=True, out="bf16", layout=2),
        # Shared key heads, blocks of 32 and odd trees over a contiguous cache.
        dict(name="tree_gqa_b5_n13", kind="tree", B=5, n_lo=1, n_hi=13, lo=33, hi=5003, bs=32,
             lb=4, K=12, H=10, Hkv=2, paged=False, out="fp32", layout=3),
        # A chain of five drafted tokens of one request against the draft's own probabilities.
        dict(name="verify_chain_b1", kind="verify", mode="chain", B=1, n_lo=6, n_hi=6, V=32000,
             type="fp32", layout=4),
        # Trees of a draft's best tokens (no draft probabilities), sampled verification.
        dict(name="verify_tree_b8_n32", kind="verify", mode="tree", B=8, n_lo=16, n_hi=32,
             V=131072, type="bf16", layout=5),
        # Trees whose siblings were sampled from the draft: one residual after another.
        dict(name="verify_siblings_b16", kind="verify", mode="siblings", B=16, n_lo=9, n_hi=24,
             V=100003, type="fp32", layout=6),
        # Greedy decoding of a serving batch: the target's best token at every node.
        dict(name="verify_greedy_b32_n48", kind="verify", mode="greedy", B=32, n_lo=24, n_hi=48,
             V=131072, type="bf16", layout=7),
        # The accepted rows of a batch moved up in the caches of 12 layers.
        dict(name="keep_b8_l12", kind="keep", B=8, n_lo=24, n_hi=64, lo=2730, hi=8190, bs=64,
             H=10, layers=12, layout=8),
        # Four prompts forked to four answers each over 12 layers, grown by a step and freed.
        dict(name="fork_b4_x4_l12", kind="fork", B=4, ways=4, lo=2730, hi=8190, bs=64, H=10,
             layers=12, grow=32, layout=9),
        # A pool of 6 layers, half of it free, compacted after its requests left.
        dict(name="compact_l6", kind="compact", B=16, lo=273, hi=2730, bs=64, H=10, layers=6,
             spare=2.0, layout=10),
        # A small pool of odd sizes.
        dict(name="compact_l1_bs32", kind="compact", B=3, lo=33, hi=999, bs=32, H=10, layers=1,
             spare=1.5, layout=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "verify", "keep", "fork", "compact"])
    layout = rng.randrange(1 << 20)
    bs, lb, K = rng.choice([(32, 4, 12), (64, 8, 8), (64, 16, 16)])
    if kind == "tree":
        hi, n = _log(rng, 20, 27300), _log(rng, 1, 64)
        return dict(kind=kind, B=_log(rng, 1, 24), n_lo=max(1, n // rng.choice([1, 2, 4])), n_hi=n,
                    lo=max(1, hi // rng.choice([1, 3, 10])), hi=hi, bs=bs, lb=lb, K=K, H=10,
                    Hkv=rng.choice([10, 10, 5, 2, 1]), paged=rng.random() < 0.7,
                    out=rng.choice(["fp32", "bf16"]), layout=layout)
    if kind == "verify":
        mode = rng.choice(["chain", "tree", "siblings", "greedy"])
        n = _log(rng, 2, 12 if mode == "chain" else 32)
        return dict(kind=kind, mode=mode, B=_log(rng, 1, 16), n_lo=max(1, n // 2), n_hi=n,
                    V=_log(rng, 300, 131072), type=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    layout=layout)
    if kind == "keep":
        n = _log(rng, 4, 64)
        return dict(kind=kind, B=_log(rng, 1, 16), n_lo=max(2, n // 2), n_hi=n,
                    lo=_log(rng, 1, 300), hi=_log(rng, 300, 8190), bs=bs,
                    H=rng.choice([10, 10, 2]), layers=rng.randrange(1, 13), layout=layout)
    if kind == "fork":
        return dict(kind=kind, B=_log(rng, 1, 8), ways=rng.randrange(1, 5), lo=_log(rng, 1, 300),
                    hi=_log(rng, 300, 8190), bs=bs, H=rng.choice([10, 10, 2]),
                    layers=rng.randrange(1, 13), grow=_log(rng, 1, 130), layout=layout)
    return dict(kind=kind, B=_log(rng, 1, 16), lo=_log(rng, 1, 270), hi=_log(rng, 270, 2730),
                bs=bs, H=rng.choice([10, 10, 2]), layers=rng.randrange(1, 7),
                spare=rng.choice([1.2, 1.5, 2.0]), layout=layout)


# ------------------------------------------------------------------------------ the inputs

def _lengths(c):
    """Context lengths and tree sizes of a case's sequences (from its layout alone, so that
    work() knows them)."""
    rng = random.Random(c["layout"] * 7919 + 11)
    lens = [rng.randint(c["lo"], c["hi"]) for _ in range(c["B"])] if "lo" in c else []
    nodes = [rng.randint(c["n_lo"], c["n_hi"]) for _ in range(c["B"])] if "n_lo" in c else []
    return lens, nodes


def _parents(rng, n, chain=False):
    """A tree in breadth-first order: a node's parent is one of the few nodes before it."""
    p = [-1] + [i - 1 if chain else max(0, (i - 1) // 3 - rng.randrange(0, 2))
                for i in range(1, n)]
    return sorted(p[:1]) + sorted(p[1:])


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).to(DEV)


def _table(rng, lens, bs, spare):
    """(block table, pool size): the pages of the sequences, taken at random from the pool."""
    need = [(n + bs - 1) // bs for n in lens]
    pool = int(math.ceil(sum(need) * spare)) + 1
    pages = rng.sample(range(pool), sum(need))
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    o = 0
    for b, m in enumerate(need):
        table[b, :m] = torch.tensor(pages[o:o + m], dtype=torch.int32)
        o += m
    return table.to(DEV), pool


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(DEV).manual_seed(seed * 1009 + 17)
    rng = random.Random(seed * 31 + c["layout"])
    s = SimpleNamespace(c=c, seed=seed)
    lens, nodes = _lengths(c)
    if nodes:
        s.cu = _i32([0] + [sum(nodes[:i + 1]) for i in range(len(nodes))])
        s.max_n = max(nodes)
        s.T = sum(nodes)
        chain = c.get("mode") == "chain"
        s.parents = _i32(sum((_parents(rng, n, chain) for n in nodes), []))
    if c["kind"] == "tree":
        _prepare_tree(s, c, g, rng, lens, nodes)
    elif c["kind"] == "verify":
        _prepare_verify(s, c, g, nodes)
    else:
        _prepare_pages(s, c, g, rng, lens, nodes)
    return s


def _prepare_tree(s, c, g, rng, lens, nodes):
    B, H, Hkv, bs, K = c["B"], c["H"], c["Hkv"], c["bs"], c["K"]
    s.ctx = _i32(lens)
    full = [a + b for a, b in zip(lens, nodes)]
    S = (max(full) + bs - 1) // bs * bs
    s.table = None
    if c["paged"]:
        s.table, pool = _table(rng, full, bs, 1.0)
        s.k = (_randn(g, pool, bs, Hkv, D) * 0.5).bfloat16()
        s.v = _randn(g, pool, bs, Hkv, D).bfloat16()
    else:
        s.k = (_randn(g, B, Hkv, S, D) * 0.5).bfloat16()
        s.v = _randn(g, B, Hkv, S, D).bfloat16()
    s.q = (_randn(g, s.T, H, D) * 0.5).bfloat16()
    # the nodes of a tree route to K of the same few blocks, as queries of one place do
    hot = [_hot(c, n) for n in lens]
    pick = torch.zeros(s.T, K, dtype=torch.int32)
    o = 0
    for b, n in enumerate(nodes):
        blocks = rng.sample(range(max(1, lens[b] // bs)), hot[b])
        for i in range(n):
            row = rng.sample(blocks, min(K, hot[b]))
            pick[o + i, :len(row)] = torch.tensor(row, dtype=torch.int32)
            pick[o + i, len(row):] = -1
        o += n
    s.idx = pick.to(DEV)
    s.bias = _randn(g, s.T, K) * 0.5
    s.valid = torch.rand(s.T, K, generator=g, device=DEV) < 0.95


def _hot(c, ctx):
    return min(2 * c["K"], max(1, ctx // c["bs"]))


def _prepare_verify(s, c, g, nodes):
    V, T, mode = c["V"], s.T, c["mode"]
    t = TYPES[c["type"]]
    base = torch.cumsum(torch.tensor([0] + nodes[:-1]), 0).to(DEV)
    seq = torch.repeat_interleave(torch.arange(len(nodes), device=DEV),
                                  torch.tensor(nodes, device=DEV))
    par = (s.parents.long().clamp(min=0) + base[seq])            # packed row of the parent
    logits = _randn(g, T, V) * 3.0
    drafted = logits + 0.7 * _randn(g, T, V)
    s.u = torch.rand(T, generator=g, device=DEV)
    s.draft = None
    same = (par[:, None] == par[None]) & (s.parents >= 0)[:, None] & (s.parents >= 0)[None]
    rank = (same & torch.ones_like(same).tril(-1)).sum(1)        # place among the siblings
    if mode in ("chain", "siblings"):
        s.draft = torch.softmax(drafted, -1).to(t)
        race = torch.empty(T, V, device=DEV).exponential_(generator=g)
        s.tokens = (torch.softmax(drafted, -1)[par] / race).argmax(-1)
    else:
        top = drafted.topk(min(V, int(rank.max()) + 1), -1).indices
        s.tokens = top[par, rank]
    s.target = (logits if mode == "greedy" else torch.softmax(logits, -1)).to(t)


def _prepare_pages(s, c, g, rng, lens, nodes):
    B, bs, H, L = c["B"], c["bs"], c["H"], c["layers"]
    if c["kind"] == "keep":
        full = [a + b for a, b in zip(lens, nodes)]
        s.table, pool = _table(rng, full, bs, 1.0)
        s.ctx = _i32(lens)
        # the root, then nodes that lie behind the places the accepted ones move to
        path = torch.full((B, s.max_n), -1, dtype=torch.int32)
        count = []
        for b, n in enumerate(nodes):
            m = rng.randint(1, max(1, min(8, n // 2)))
            rows = [0] + sorted(rng.sample(range(m, n), m - 1))
            path[b, :m] = torch.tensor(rows, dtype=torch.int32)
            count.append(m)
        s.path, s.count = path.to(DEV), _i32(count)
    elif c["kind"] == "fork":
        ways, grow = c["ways"], c["grow"]
        rows = B * (1 + ways)
        need = [(n + bs - 1) // bs for n in lens]
        new = [(n + grow + bs - 1) // bs - n // bs for n in lens]
        P = max(need) + (grow + bs - 1) // bs + 1
        table, pool = _table(rng, lens, bs, 1.0)
        pool += ways * sum(new) + 3
        s.table = torch.full((rows, P), -1, dtype=torch.int32, device=DEV)
        s.table[:B, :table.shape[1]] = table
        s.lens = torch.zeros(rows, dtype=torch.int32, device=DEV)
        s.lens[:B] = _i32(lens)
        s.src = _i32([b for b in range(B) for _ in range(ways)])
        s.dst = _i32(list(range(B, rows)))
        s.new_lens = s.lens.clone()
        s.new_lens[B:] = s.lens[s.src.long()] + grow
        s.keep_lens = s.lens.clone()
    else:
        s.table, pool = _table(rng, lens, bs, c["spare"])
        s.lens = _i32(lens)
    if c["kind"] != "keep":
        used = s.table[s.table >= 0].long()
        s.refs = torch.zeros(pool, dtype=torch.int32, device=DEV).index_add_(
            0, used, torch.ones_like(used, dtype=torch.int32))
    s.k = _randn(g, L, pool, bs, H, D).bfloat16()
    s.v = _randn(g, L, pool, bs, H, D).bfloat16()
    s.idx_k = _randn(g, L, pool, bs, D)


# ------------------------------------------------------------------------------ one pass

def run(s):
    c = s.c
    if own:
        return _run_own(s, c)
    return {"tree": _plain_tree, "verify": _plain_verify, "keep": _plain_keep,
            "fork": _plain_fork, "compact": _plain_compact}[c["kind"]](s, c)


def _run_own(s, c):
    from ananta_ocr_amd import kv_pages, tree
    kind = c["kind"]
    if kind == "tree":
        mask, depth = tree.tree_masks(s.parents, s.cu, s.max_n)
        out = tree.attn_tree(s.q, s.k, s.v, s.idx, s.bias, s.valid, mask, depth, s.ctx, s.cu,
                             s.max_n, c["bs"], c["lb"] * c["bs"], SCALE, block_table=s.table,
                             page_size=c["bs"], out_dtype=TYPES[c["out"]])
        return out, depth
    if kind == "verify":
        return tree.verify_tree(s.target, s.tokens, s.parents, s.cu, s.max_n,
                                uniforms=None if c["mode"] == "greedy" else s.u, draft=s.draft)
    caches = kv_pages.PageCaches([s.k, s.v, s.idx_k], layered=True)
    if kind == "keep":
        kv_pages.keep_rows(caches, s.path, s.count, s.ctx, s.table)
        return s.k, s.v, s.idx_k
    if kind == "fork":
        ok, frm, to = kv_pages.fork_pages(s.refs, s.table, s.lens, s.src, s.dst, c["bs"])
        kv_pages.copy_pages(caches, frm, to)
        ok2, frm2, to2 = kv_pages.reserve_pages(s.refs, s.table, s.lens, s.new_lens, c["bs"])
        kv_pages.copy_pages(caches, frm2, to2)
        grown = s.table.clone(), s.refs.clone()
        kv_pages.free_pages(s.refs, s.table, s.lens, s.keep_lens, c["bs"])
        return ok, frm, to, ok2, frm2, to2, grown, s.table, s.refs, s.lens, s.k, s.v, s.idx_k
    refs, table, frm, to = kv_pages.compact_pages(s.refs, s.table, s.lens, c["bs"])
    kv_pages.copy_pages(caches, frm, to)
    return refs, table, frm, to, s.k, s.v, s.idx_k


# ------------------------------------------------------------------------------ plain forms

def _rows(s):
    """Sequence and node of every packed row, and the packed row of its parent (-1: none)."""
    n = (s.cu[1:] - s.cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=s.T)
    base = s.cu[:-1].long()[seq]
    node = torch.arange(s.T, device=DEV) - base
    return seq, node, base, torch.where(s.parents >= 0, s.parents.long() + base, -1)


def _closure(par):
    """[T, T] whether column j is row i or one of its ancestors."""
    T = par.numel()
    step = (par[:, None] == torch.arange(T, device=DEV)[None]) | torch.eye(
        T, dtype=torch.bool, device=DEV)
    return torch.linalg.matrix_power(step.double(), T) > 0.5


def _plain_tree(s, c):
    B, H, Hkv, bs, K = c["B"], c["H"], c["Hkv"], c["bs"], c["K"]
    lw, N, G = c["lb"] * bs, s.max_n, H // Hkv
    seq, node, base, par = _rows(s)
    anc = _closure(par)
    depth = (anc.sum(1) - 1).to(torch.int32)
    if s.table is not None:
        pages = s.table.long().clamp(min=0)
        k = s.k[pages].reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float()
        v = s.v[pages].reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float()
    else:
        k, v = s.k.float(), s.v.float()
    S = k.shape[2]
    ctx = s.ctx.long()[seq][:, None]
    first = ctx + depth[:, None] - lw + 1                     # first window position of a row
    j = torch.arange(S, device=DEV)[None]
    nblk = (S + bs - 1) // bs
    # routed blocks: valid, below the window, a block's first slot
    ok = s.valid & (s.idx >= 0) & (s.idx < nblk) & (s.idx * bs < torch.minimum(first, ctx))
    same = (s.idx[:, :, None] == s.idx[:, None, :]) & ok[:, None, :]
    ok &= ~(same & torch.ones(K, K, dtype=torch.bool, device=DEV).tril(-1)).any(-1)
    at = torch.where(ok, s.idx, nblk).long()
    named = torch.zeros(s.T, nblk + 1, device=DEV).scatter_(1, at, 1.0)[:, :nblk] > 0
    extra = torch.zeros(s.T, nblk + 1, device=DEV).scatter_(1, at, s.bias)[:, :nblk]
    named = named.repeat_interleave(bs, 1)[:, :S]
    extra = extra.repeat_interleave(bs, 1)[:, :S]
    remote = named & (j < first) & (j < ctx)
    slot = (j - ctx).clamp(0, N - 1)
    drafted = torch.zeros(s.T, N, dtype=torch.bool, device=DEV)
    drafted[torch.arange(s.T, device=DEV)[:, None].expand_as(anc)[anc], node[None].expand_as(anc)[anc]] = True
    sees = remote | ((j >= first) & (j < ctx)) | (
        (j >= ctx) & (j < ctx + N) & drafted.gather(1, slot))
    add = torch.where(sees, torch.where(remote, extra, 0.0), -math.inf)
    q = torch.zeros(B, N, H, D, device=DEV)
    q[seq, node] = s.q.float()
    bias = torch.zeros(B, N, S, device=DEV)
    bias[seq, node] = add
    q = q.view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hkv, G, N, S)
    z = z * SCALE + bias[:, None, None]
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, G * N, S), v).view(B, Hkv, G, N, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, H, D)[seq, node]
    return o.to(TYPES[c["out"]]), depth


def _plain_verify(s, c):
    B, N, V, T = c["B"], s.max_n, c["V"], s.T
    seq, node, base, par = _rows(s)
    child = par >= 0
    up = par.clamp(min=0)
    tok = s.tokens.long()
    same = (par[:, None] == par[None]) & child[:, None] & child[None]
    before = same & torch.ones_like(same).tril(-1)           # earlier siblings
    i = torch.arange(T, device=DEV)
    gone = torch.zeros(T, device=DEV, dtype=torch.float64)   # a node's rejected draft share
    if c["mode"] == "greedy":
        t = s.target.float()
        best = torch.where(t == t.amax(-1, keepdim=True), torch.arange(V, device=DEV), V).amin(-1)
        match = child & (tok == best[up])
        yes = match & ~(before & match[None]).any(1)
    elif s.draft is None:
        p = s.target.double()
        again = (before & (tok[:, None] == tok[None])).any(1)
        e = torch.where(child & ~again, p[up, tok], 0.0)
        yes = s.u.double() * (1.0 - before.double() @ e) < e
        yes &= ~(before & yes[None]).any(1)
    else:
        p, q = s.target.double(), s.draft.double()
        left = torch.ones_like(gone)                         # a node's remaining mass
        rank = before.sum(1)
        yes = torch.zeros(T, dtype=torch.bool, device=DEV)
        for r in range(int(rank.max()) + 1):
            mine = child & (rank == r)
            y = s.u.double() * left[up] * q[up, tok] < (p[up, tok] - gone[up] * q[up, tok]).clamp(
                min=0)
            yes |= mine & y
            lost = torch.zeros(T, dtype=torch.bool, device=DEV)
            lost[up[mine & ~y]] = True
            gone = torch.where(lost, gone + left, gone)
            left = torch.where(lost, (p - gone[:, None] * q).clamp(min=0).sum(-1), left)
        yes &= ~(before & yes[None]).any(1)
    anc = _closure(par)
    on = ~(anc & child[None] & ~yes[None]).any(1)            # every step from the root accepted
    count = torch.zeros(B, dtype=torch.int32, device=DEV).index_add_(0, seq, on.to(torch.int32))
    depth = anc.sum(1) - 1
    path = torch.full((B, N), -1, dtype=torch.int32, device=DEV)
    path[seq[on], depth[on]] = node[on].to(torch.int32)
    last = torch.zeros(B, dtype=torch.long, device=DEV).scatter_reduce_(
        0, seq, torch.where(on, i, 0), "amax")                # the deepest accepted node
    if c["mode"] == "greedy":
        return count, path, best[last]
    r = s.target[last].double()
    if s.draft is not None:
        r = (r - gone[last][:, None] * s.draft[last].double()).clamp(min=0)
    else:
        kids = child & (last[seq] == par)
        r[seq[kids], tok[kids]] = 0.0
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, s.target[last].double())
    sums = r.cumsum(-1)
    over = sums > s.u[s.cu[:-1].long()].double()[:, None] * sums[:, -1:]
    v = torch.arange(V, device=DEV)
    token = torch.where(over, v, V).amin(-1)
    return count, path, torch.where(token < V, token, torch.where(r > 0, v, -1).amax(-1))


def _plain_keep(s, c):
    bs = c["bs"]
    at = torch.arange(s.max_n, device=DEV)[None]
    moved = (at < s.count[:, None]) & (s.path != at)
    b = torch.arange(c["B"], device=DEV)[:, None].expand_as(moved)[moved]
    frm = (s.ctx[:, None] + s.path)[moved].long()
    to = (s.ctx[:, None] + at)[moved].long()
    fp, tp = s.table[b, frm // bs].long(), s.table[b, to // bs].long()
    for x in (s.k, s.v, s.idx_k):
        x[:, tp, to % bs] = x[:, fp, frm % bs]
    return s.k, s.v, s.idx_k


def _copy(s, frm, to):
    f, t = frm[frm >= 0].long(), to[to >= 0].long()
    for x in (s.k, s.v, s.idx_k):
        x[:, t] = x[:, f]


def _plain_fork(s, c):
    bs = c["bs"]
    src, dst = s.src.long(), s.dst.long()
    P = s.table.shape[1]
    at = torch.arange(P, device=DEV)[None]
    n = s.lens[src]
    full = at < (n // bs)[:, None]
    pages = s.table[src]
    s.refs.index_add_(0, pages[full].long(), torch.ones_like(pages[full]))
    row = torch.where(full, pages, -1)
    tail = n % bs > 0
    where = torch.arange(s.refs.numel(), device=DEV)
    order = torch.sort(torch.where(s.refs == 0, where, s.refs.numel())).values   # free, lowest first
    new = order[(tail.long().cumsum(0) - 1).clamp(min=0)].to(torch.int32)
    frm = torch.where(tail, pages.gather(1, (n // bs).long()[:, None])[:, 0], -1)
    to = torch.where(tail, new, -1)
    row = torch.where((at == (n // bs)[:, None]) & tail[:, None], to[:, None], row)
    s.table[dst] = row
    s.refs.index_add_(0, to[tail].long(), torch.ones_like(to[tail]))
    s.lens[dst] = n
    _copy(s, frm, to)
    # growth: whole new pages, rows in order (a forked row's tail page is its own)
    have, want = (s.lens + bs - 1) // bs, (s.new_lens + bs - 1) // bs
    need = (at >= have[:, None]) & (at < want[:, None])
    order = torch.sort(torch.where(s.refs == 0, where, s.refs.numel())).values
    s.table[need] = order[:int(need.sum())].to(torch.int32)
    got = s.table[need]
    s.refs.index_add_(0, got.long(), torch.ones_like(got))
    s.lens.copy_(torch.maximum(s.lens, s.new_lens))
    none = torch.full_like(s.lens, -1)
    grown = s.table.clone(), s.refs.clone()
    # the children leave
    drop = at >= ((s.keep_lens + bs - 1) // bs)[:, None]
    drop = drop & (s.table >= 0)
    out = s.table[drop]
    s.refs.index_add_(0, out.long(), -torch.ones_like(out))
    s.table[drop] = -1
    s.lens.copy_(torch.minimum(s.lens, s.keep_lens))
    ok = torch.ones(1, dtype=torch.int32, device=DEV)
    return (ok, frm, to, ok.clone(), none, none.clone(), grown, s.table, s.refs, s.lens, s.k, s.v,
            s.idx_k)


def _plain_compact(s, c):
    n = s.refs.numel()
    where = torch.arange(n, device=DEV)
    live = s.refs > 0
    total = live.sum()
    high, low = live & (where >= total), ~live & (where < total)
    rank = torch.zeros(n, dtype=torch.long, device=DEV)
    slot = torch.full((n + 1,), -1, dtype=torch.long, device=DEV)
    slot[torch.where(low, low.long().cumsum(0) - 1, n)] = where
    slot[n] = -1
    rank = (high.long().cumsum(0) - 1).clamp(min=0)
    to_of = torch.where(high, slot[rank], where)
    refs = torch.zeros_like(s.refs)
    refs[to_of[live]] = s.refs[live]
    table = torch.where(s.table >= 0, to_of[s.table.clamp(min=0).long()].to(torch.int32), -1)
    frm = torch.full((n // 2 + 1,), -1, dtype=torch.int32, device=DEV)
    to = frm.clone()
    m = torch.where(high, rank, n // 2)
    frm[m] = where.to(torch.int32)
    to[m] = to_of.to(torch.int32)
    frm, to = frm[:n // 2], to[:n // 2]
    last = torch.arange(n // 2, device=DEV) < high.sum()
    frm, to = torch.where(last, frm, -1), torch.where(last, to, -1)
    _copy(s, frm, to)
    return refs, table, frm, to, s.k, s.v, s.idx_k


# ------------------------------------------------------------------------------ exact

def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    kind = c["kind"]
    if kind == "tree":
        return _exact_tree(s, c)
    if kind == "verify":
        return _exact_verify(s, c)
    return _exact_pages(s, c)


def _exact_tree(s, c):
    """Row by row of every sequence, its keys listed one set after another."""
    H, Hkv, bs, lw = c["H"], c["Hkv"], c["bs"], c["lb"] * c["bs"]
    cu, ctx, par = s.cu.tolist(), s.ctx.tolist(), s.parents.tolist()
    idx, valid = s.idx.tolist(), s.valid.tolist()
    table = None if s.table is None else s.table.tolist()
    out, depths = [], []
    for b in range(c["B"]):
        n, S = cu[b + 1] - cu[b], ctx[b] + cu[b + 1] - cu[b]
        if table is not None:
            pg = torch.tensor(table[b][:(S + bs - 1) // bs], device=DEV)
            k, v = (x[pg].reshape(-1, Hkv, D)[:S].double() for x in (s.k, s.v))
        else:
            k, v = (x[b, :, :S].transpose(0, 1).double() for x in (s.k, s.v))
        z = torch.full((n, H, S), -math.inf, dtype=torch.float64)
        z = z.to(DEV)
        chains = []
        for i in range(n):
            up, chain = i, []
            while up >= 0:
                chain.append(up)
                up = par[cu[b] + up]
            chains.append(chain)
        depths += [len(x) - 1 for x in chains]
        dots = torch.stack([s.q[cu[b]:cu[b + 1], h].double() @ k[:, h // (H // Hkv)].t().contiguous()
                            for h in range(H)], 1) * SCALE            # [n, H, S]
        for i in range(n):
            r = cu[b] + i
            w0 = ctx[b] + len(chains[i]) - 1 - lw + 1
            cols = list(range(max(w0, 0), ctx[b])) + [ctx[b] + m for m in chains[i]]
            extra = torch.zeros(S, dtype=torch.float64)
            bias = s.bias[r].tolist()
            done = set()
            for x, ok, y in zip(idx[r], valid[r], bias):
                if not ok or x < 0 or x in done:
                    continue
                some = range(x * bs, min((x + 1) * bs, w0, ctx[b]))
                if len(some):
                    done.add(x)
                    cols += list(some)
                    extra[x * bs:some[-1] + 1] = y
            at = torch.tensor(cols, device=DEV)
            z[i][:, at] = dots[i][:, at] + extra.to(DEV)[at][None]
        p = torch.softmax(z, -1)
        out.append(torch.stack([p[:, h] @ v[:, h // (H // Hkv)].contiguous() for h in range(H)], 1))
    return torch.cat(out), torch.tensor(depths, dtype=torch.int32)


def _exact_verify(s, c):
    """The walk from every root, by Python's own floats."""
    V, mode = c["V"], c["mode"]
    cu, par, tok = s.cu.tolist(), s.parents.tolist(), s.tokens.tolist()
    u = s.u.double().tolist()
    counts, paths, tokens = [], [], []
    for b in range(c["B"]):
        n, at, path = cu[b + 1] - cu[b], 0, [0]
        while True:
            row = s.target[cu[b] + at].double().cpu()
            kids = [i for i in range(1, n) if par[cu[b] + i] == at]
            if mode == "greedy":
                best = min((row == row.max()).nonzero().flatten().tolist())
                hit = [i for i in kids if tok[cu[b] + i] == best]
                if not hit:
                    tokens.append(best)
                    break
                at = hit[0]
                path.append(at)
                continue
            q = None if s.draft is None else s.draft[cu[b] + at].double().cpu()
            rest, mass, found = row.clone(), 1.0, None
            for i in kids:
                x = tok[cu[b] + i]
                share = 1.0 if q is None else float(q[x])
                if u[cu[b] + i] * mass * share < float(rest[x]):
                    found = i
                    break
                if q is None:
                    mass -= float(rest[x])
                    rest[x] = 0.0
                else:
                    rest = (rest - mass * q).clamp(min=0)
                    mass = float(rest.sum())
            if found is not None:
                at = found
                path.append(at)
                continue
            rest = rest if float(rest.sum()) > 0 else row
            run_ = rest.cumsum(0)
            over = (run_ > u[cu[b]] * run_[-1]).nonzero()
            tokens.append(int(over[0]) if len(over) else int((rest > 0).nonzero()[-1]))
            break
        counts.append(len(path))
        paths.append(path + [-1] * (s.max_n - len(path)))
    return (torch.tensor(counts, dtype=torch.int32), torch.tensor(paths, dtype=torch.int32),
            torch.tensor(tokens))


def _exact_pages(s, c):
    """The caches by moves of single pages and rows, the tables by lists."""
    bs = c["bs"]
    if c["kind"] == "keep":
        ctx, table = s.ctx.tolist(), s.table.tolist()
        for b, (path, m) in enumerate(zip(s.path.tolist(), s.count.tolist())):
            old = [(ctx[b] + x) for x in path[:m]]
            for x in (s.k, s.v, s.idx_k):
                rows = [x[:, table[b][o // bs], o % bs].clone() for o in old]
                for i, r in enumerate(rows):
                    o = ctx[b] + i
                    x[:, table[b][o // bs], o % bs] = r
        return s.k.double(), s.v.double(), s.idx_k.double()
    refs, table, lens = s.refs.tolist(), s.table.tolist(), s.lens.tolist()

    def move(a, b):
        for x in (s.k, s.v, s.idx_k):
            x[:, b] = x[:, a].clone()

    def ints(x):
        return torch.tensor(x, dtype=torch.int32)

    if c["kind"] == "fork":
        frm, to = [], []
        before = [list(r) for r in table], list(refs), list(lens)
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            for i in range(lens[a] // bs):
                table[b][i] = table[a][i]
                refs[table[a][i]] += 1
            frm.append(-1)
            to.append(-1)
            if lens[a] % bs:
                i = lens[a] // bs
                new = refs.index(0)
                refs[new], table[b][i] = 1, new
                frm[-1], to[-1] = table[a][i], new
                move(table[a][i], new)
            lens[b] = lens[a]
        for b, n in enumerate(s.new_lens.tolist()):
            for i in range((lens[b] + bs - 1) // bs, (n + bs - 1) // bs):
                new = refs.index(0)
                refs[new], table[b][i] = 1, new
        none = ints([-1] * len(lens))
        # freed, the tables are what they were
        return (ints([1]), ints(frm), ints(to), ints([1]), none, none, (ints(table), ints(refs)),
                ints(before[0]), ints(before[1]), ints(before[2]), s.k.double(), s.v.double(),
                s.idx_k.double())
    total = sum(r > 0 for r in refs)
    frm, to, place = [], [], {}
    for i in range(total, len(refs)):
        if refs[i]:
            new = next(x for x in range(total) if refs[x] == 0)
            refs[new], refs[i] = refs[i], 0
            place[i] = new
            frm.append(i)
            to.append(new)
            move(i, new)
    pad = [-1] * (len(refs) // 2 - len(frm))
    return (ints(refs), ints([[place.get(x, x) for x in r] for r in table]), ints(frm + pad),
            ints(to + pad), s.k.double(), s.v.double(), s.idx_k.double())


# ------------------------------------------------------------------------------ the work

def work(case):
    c = dict(case)
    lens, nodes = _lengths(c)
    if c["kind"] == "tree":
        bs, lw = c["bs"], c["lb"] * c["bs"]
        rows = sum(nodes)
        # the window, the drafted keys and the blocks a tree's nodes name, once each for a head
        keys = sum(min(n, lw) + m + min(_hot(c, n) * bs, max(n - lw, 0))
                   for n, m in zip(lens, nodes))
        seen = sum(m * (min(n, lw) + min(c["K"] * bs, max(n - lw, 0)) + m / 4)
                   for n, m in zip(lens, nodes))
        out = 2 if c["out"] == "bf16" else 4
        return {"bytes": keys * c["Hkv"] * D * 4 + rows * c["H"] * D * (2 + out)
                + rows * c["K"] * 9 + rows * 12, "flops": 4.0 * seen * c["H"] * D}
    if c["kind"] == "verify":
        size = 4 if c["type"] == "fp32" else 2
        V, rows = c["V"], sum(nodes)
        if c["mode"] == "greedy":
            return {"bytes": rows * (V * size + 12), "flops": rows * V}
        # the last node's row (and the draft's) once to sum and once to draw from
        both = 1 if c["mode"] == "tree" else 2
        return {"bytes": c["B"] * V * size * both + rows * 24, "flops": 4 * c["B"] * V * both}
    row = c["H"] * D * 4 + D * 4                             # K, V and index key of a token
    L = c["layers"]
    if c["kind"] == "keep":
        # up to 8 rows of a tree, 4 or 5 as a rule, read and written
        moved = sum(max(0.5, (min(8, n // 2) - 1) / 2) for n in nodes)
        return {"bytes": 2 * moved * row * L + c["B"] * 40, "flops": 1}
    if c["kind"] == "fork":
        tails = c["ways"] * sum(n % c["bs"] > 0 for n in lens)
        pages = sum((n + c["bs"] - 1) // c["bs"] for n in lens)
        return {"bytes": 2 * tails * c["bs"] * row * L + 16 * pages * (1 + c["ways"]), "flops": 1}
    pages = sum((n + c["bs"] - 1) // c["bs"] for n in lens)
    pool = int(math.ceil(pages * c["spare"])) + 1
    moved = pages * (pool - pages) / pool                    # those that lie above the live count
    return {"bytes": 2 * moved * c["bs"] * row * L + 8 * (pool + pages), "flops": 1}
