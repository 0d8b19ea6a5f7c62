"""Measured cases of the operators that serve several answers to one prompt over a paged cache: where
the new tokens of every request go (``rows``), their rotary positions, alone with a backward pass
(``turn``) or together with the write of their keys and values (``append``), full attention that
reads a prompt once for all of its answers (``shared``), and the next token drawn from the logits,
with the probabilities that a verification takes (``sample``).

Heads (10), head dim (128), pages of 64 tokens and prompts of 10 to 100 pages of 273 tokens are
those of the checkpoint's configuration and of the benchmark.  Vocabularies are generic.
"""

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------ the cases

def listed():
    return [
        # A decode step of eight requests in a batch of a fixed size.
        dict(name="rows_b8", kind="rows", B=8, n_lo=1, n_hi=1, lo=2730, hi=27300, bs=64, spare=8,
             layout=0),
        # Prompts in chunks beside decode rows: 256 requests, none to two document pages each.
        dict(name="rows_b256", kind="rows", B=256, n_lo=0, n_hi=546, lo=0, hi=8190, bs=64,
             spare=100, layout=1),
        # The new tokens of eight requests, rotated and written to their pages.
        dict(name="append_t8", kind="append", T=8, lo=2730, hi=27300, bs=64, H=10, Hkv=10, rot=128,
             start=0, pairs=False, far=1.0, type="bf16", layout=2),
        # A prompt of 30 pages of 273 tokens, positions scaled for long contexts.
        dict(name="append_t8190", kind="append", T=8190, lo=0, hi=0, bs=64, H=10, Hkv=10, rot=128,
             start=0, pairs=False, far=40.0, type="bf16", layout=3),
        # Training: the last half of every head by interleaved pairs, and the gradients.
        dict(name="turn_b2_s4095", kind="turn", B=2, S=4095, H=10, Hkv=10, rot=64, start=64,
             pairs=True, far=1.0, type="bf16", layout=4),
        # Four answers to a prompt of ten pages: latency.
        dict(name="shared_g1_b4", kind="shared", G=1, w_lo=4, w_hi=4, n_lo=1, n_hi=1, p_lo=2730,
             p_hi=2730, o_lo=1, o_hi=64, bs=64, H=10, Hkv=10, out="fp32", layout=5),
        # Four long documents with a few answers each.
        dict(name="shared_g4_b32", kind="shared", G=4, w_lo=4, w_hi=12, n_lo=1, n_hi=1, p_lo=8190,
             p_hi=27300, o_lo=1, o_hi=600, bs=64, H=10, Hkv=10, out="bf16", layout=6),
        # One document of 100 pages, 64 answers of up to 1,000 tokens.
        dict(name="shared_g1_b64", kind="shared", G=1, w_lo=64, w_hi=64, n_lo=1, n_hi=1,
             p_lo=27300, p_hi=27300, o_lo=1, o_hi=1000, bs=64, H=10, Hkv=10, out="bf16", layout=7),
        # Shared key heads, several rows a request, small pages, odd lengths.
        dict(name="shared_gqa_g3_b9", kind="shared", G=3, w_lo=1, w_hi=5, n_lo=1, n_hi=7, p_lo=0,
             p_hi=5003, o_lo=0, o_hi=333, bs=16, H=10, Hkv=2, out="fp32", layout=8),
        # One request, a small vocabulary.
        dict(name="sample_b1_v32000", kind="sample", R=1, V=32000, type="fp32", probs=False,
             layout=9),
        # A serving batch, a large vocabulary.
        dict(name="sample_b64_v131072", kind="sample", R=64, V=131072, type="bf16", probs=False,
             layout=10),
        # The target's probabilities of a batch of drafted tokens, as a verification takes them.
        dict(name="probs_b48_v100003", kind="sample", R=48, V=100003, type="fp32", probs=True,
             layout=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "append", "turn", "shared", "shared", "sample", "sample"])
    c = dict(kind=kind, layout=rng.randrange(1 << 20))
    heads = dict(H=10, Hkv=rng.choice([10, 10, 5, 2, 1]))
    bs = rng.choice([16, 32, 64, 64, 128])
    if kind == "rows":
        n = _log(rng, 1, 546)
        return dict(c, B=_log(rng, 1, 256), n_lo=rng.choice([0, 1]), n_hi=n, lo=0,
                    hi=_log(rng, 1, 8190), bs=bs, spare=rng.randrange(0, 200))
    rot = rng.choice([128, 128, 64, 32])
    turn = dict(rot=rot, start=rng.choice([0, D - rot]), pairs=rng.random() < 0.5,
                far=rng.choice([1.0, 4.0, 40.0]), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "append":
        lo = rng.choice([0, _log(rng, 1, 27300)])
        return dict(c, T=_log(rng, 1, 8190), lo=lo, hi=lo + rng.choice([0, 8190]), bs=bs, **heads,
                    **turn)
    if kind == "turn":
        return dict(c, B=rng.randrange(1, 3), S=_log(rng, 1, 4095), **heads, **turn)
    if kind == "shared":
        ways, p, o = _log(rng, 1, 24), _log(rng, 1, 27300), _log(rng, 1, 1000)
        n = _log(rng, 1, 16)
        return dict(c, G=rng.randrange(1, 4 if p < 10000 else 3), w_lo=max(1, ways // 2), w_hi=ways,
                    n_lo=max(1, n // 2), n_hi=n, p_lo=rng.choice([0, p // 2, p]), p_hi=p,
                    o_lo=rng.choice([0, 1]), o_hi=o, bs=bs, out=rng.choice(["fp32", "bf16"]),
                    **heads)
    return dict(c, R=_log(rng, 1, 48), V=_log(rng, 300, 131072), probs=rng.random() < 0.4,
                type=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


# ------------------------------------------------------------------------------ the inputs

def _lengths(c):
    """What a case's lengths are, from its layout alone, so that work() knows them: for requests
    their contexts and new rows, for groups also the prompts and the number of answers."""
    rng = random.Random(c["layout"] * 7919 + 11)
    if c["kind"] == "rows":
        ctx = [rng.randint(c["lo"], c["hi"]) for _ in range(c["B"])]
        return ctx, [rng.randint(c["n_lo"], c["n_hi"]) for _ in ctx], None, None
    ways = [rng.randint(c["w_lo"], c["w_hi"]) for _ in range(c["G"])]
    # whole pages of a prompt are shared; the rest of it lies in every answer's own pages
    prompts = [rng.randint(c["p_lo"], c["p_hi"]) for _ in ways]
    ctx, new = [], []
    for w, p in zip(ways, prompts):
        ctx += [p + rng.randint(c["o_lo"], c["o_hi"]) for _ in range(w)]
        new += [rng.randint(c["n_lo"], c["n_hi"]) for _ in range(w)]
    return ctx, new, ways, [p // c["bs"] * c["bs"] for p in prompts]


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).to(DEV)


def _sums(x):
    out = [0]
    for n in x:
        out.append(out[-1] + n)
    return out


def _table(rng, ctx, new, ways, shared, bs):
    """(block table, pool size): pages taken at random, the first ones of a group in common."""
    need = [(a + b + bs - 1) // bs for a, b in zip(ctx, new)]
    pool = sum(need) + 3
    free = rng.sample(range(pool), pool)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32)
    b = 0
    for w, p in zip(ways, shared):
        first = [free.pop() for _ in range(p // bs)]
        for b in range(b, b + w):
            row = first + [free.pop() for _ in range(need[b] - len(first))]
            table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        b += 1
    return table.to(DEV), pool


def _inv_freq(c):
    """(angular frequencies [rot / 2] in 64 bits, factor of cos and sin).  far > 1: low frequencies
    are divided by it, high ones kept, with a ramp between 32 and 1 turns over 4,096 positions."""
    m, base, far = c["rot"] // 2, 10000.0, c["far"]
    f = torch.tensor([base ** (-j / m) for j in range(m)], dtype=torch.float64)
    if far == 1.0:
        return f, 1.0

    def at(turns):
        return m * math.log(4096 / (turns * 2 * math.pi)) / math.log(base)

    lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), m - 1)
    ramp = ((torch.arange(m, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f / far * ramp + f * (1 - ramp), 0.1 * math.log(far) + 1.0


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(DEV).manual_seed(seed * 1009 + 17)
    rng = random.Random(seed * 31 + c["layout"])
    s = SimpleNamespace(c=c, seed=seed)
    {"rows": _prepare_rows, "append": _prepare_append, "turn": _prepare_turn,
     "shared": _prepare_shared, "sample": _prepare_sample}[c["kind"]](s, c, g, rng)
    return s


def _prepare_rows(s, c, g, rng):
    ctx, new, _, _ = _lengths(c)
    order = rng.sample(range(len(ctx)), len(ctx))
    ctx, new = [ctx[i] for i in order], [new[i] for i in order]
    s.table, s.pool = _table(rng, ctx, new, [1] * len(ctx), [0] * len(ctx), c["bs"])
    s.ctx, s.new = _ints(ctx), _ints(new)
    s.rows = sum(new) + c["spare"]


def _qkv(s, c, g, lead):
    """Queries, keys and values as one projection leaves them."""
    H, Hkv = c["H"], c["Hkv"]
    x = _randn(g, *lead, (H + 2 * Hkv) * D).to(TYPES[c["type"]])
    x = x.view(*lead, H + 2 * Hkv, D)
    s.q, s.k, s.v = x.split((H, Hkv, Hkv), -2)


def _prepare_append(s, c, g, rng):
    T, bs = c["T"], c["bs"]
    _qkv(s, c, g, (T,))
    pages = (T + bs - 1) // bs + 2
    if c["hi"] > c["lo"]:                                    # tokens of many requests
        pages = 2 * pages
        pos = [rng.randint(c["lo"], c["hi"]) for _ in range(T)]
        slots = rng.sample(range(pages * bs), T)
    else:                                                    # one request's, one after another
        pos = list(range(c["lo"], c["lo"] + T))
        order = rng.sample(range(pages), pages)
        slots = [order[i // bs] * bs + i % bs for i in range(T)]
    s.pos, s.slots = _ints(pos), _ints(slots, torch.int64)
    s.k_cache = _randn(g, pages, bs, c["Hkv"], D).to(TYPES[c["type"]])
    s.v_cache = _randn(g, pages, bs, c["Hkv"], D).to(TYPES[c["type"]])
    f, s.factor = _inv_freq(c)
    s.inv_freq = f.to(DEV)


def _prepare_turn(s, c, g, rng):
    B, S = c["B"], c["S"]
    _qkv(s, c, g, (B, S))
    # documents start anywhere in a longer one
    s.pos = _ints([[a + i for i in range(S)] for a in (rng.randint(0, 8190) for _ in range(B))])
    s.dq = _randn(g, B, S, c["H"], D).to(TYPES[c["type"]])
    s.dk = _randn(g, B, S, c["Hkv"], D).to(TYPES[c["type"]])
    f, s.factor = _inv_freq(c)
    s.inv_freq = f.to(DEV)
    s.q, s.k = s.q.detach().requires_grad_(), s.k.detach().requires_grad_()


def _prepare_shared(s, c, g, rng):
    ctx, new, ways, shared = _lengths(c)
    s.lens = ctx, new, ways, shared
    s.table, pool = _table(rng, ctx, new, ways, shared, c["bs"])
    s.ctx, s.cu = _ints(ctx), _ints(_sums(new))
    s.cu_groups, s.prefix = _ints(_sums(ways)), _ints(shared)
    s.q = (_randn(g, sum(new), c["H"], D) * 0.7).bfloat16()
    s.k_cache = (_randn(g, pool, c["bs"], c["Hkv"], D) * 0.7).bfloat16()
    s.v_cache = _randn(g, pool, c["bs"], c["Hkv"], D).bfloat16()


def _prepare_sample(s, c, g, rng):
    R, V = c["R"], c["V"]
    x = 2.5 * _randn(g, R, V)
    # a few tokens stand out, and the vocabulary's padding is masked
    at = torch.randint(0, V, (R, 24), generator=g, device=DEV)
    x.scatter_add_(1, at, 6.0 * torch.rand(R, 24, generator=g, device=DEV) + 3.0)
    x[:, V - V // 100:] = -math.inf
    s.logits = x.to(TYPES[c["type"]])
    s.u = torch.rand(R, generator=g, device=DEV)
    # every request has its own settings; a temperature of 0 takes the best token
    pick = [(rng.choice([0.0] + 7 * [round(rng.uniform(0.3, 1.3), 2)]),
             rng.choice([0, 0, 1, 20, 50, 200, 1000]), rng.choice([1.0, 0.8, 0.9, 0.95, 0.98]),
             rng.choice([0.0, 0.0, 0.02, 0.1])) for _ in range(R)]
    t, k, p, m = zip(*pick)
    s.temperature, s.top_k = torch.tensor(t).to(DEV), _ints(k)
    s.top_p, s.min_p = torch.tensor(p).to(DEV), torch.tensor(m).to(DEV)


# ------------------------------------------------------------------------------ one pass

def run(s):
    c = s.c
    if own:
        return _run_own(s, c)
    return {"rows": _plain_rows, "append": _plain_append, "turn": _plain_turn,
            "shared": _plain_shared, "sample": _plain_sample}[c["kind"]](s, c)


def _run_own(s, c):
    from ananta_ocr_amd import kv_pages, rope, sampling, shared_prefix
    kind = c["kind"]
    if kind == "rows":
        return kv_pages.step_rows(s.table, s.ctx, s.new, c["bs"], s.pool, s.rows)
    if kind == "append":
        q = rope.rope_append(s.q, s.k, s.v, s.pos, s.slots, s.k_cache, s.v_cache, s.inv_freq,
                             interleaved=c["pairs"], start=c["start"], factor=s.factor)
        return q, s.k_cache, s.v_cache
    if kind == "turn":
        q, k = rope.apply_rope(s.q, s.k, s.pos, s.inv_freq, interleaved=c["pairs"],
                               start=c["start"], factor=s.factor)
        dq, dk = torch.autograd.grad((q, k), (s.q, s.k), (s.dq, s.dk))
        return q.detach(), k.detach(), dq, dk
    if kind == "shared":
        return shared_prefix.attn_shared(s.q, s.k_cache, s.v_cache, s.table, s.ctx, s.cu,
                                         s.cu_groups, s.prefix, SCALE, out_dtype=TYPES[c["out"]])
    return sampling.sample(s.logits, s.u, s.temperature, s.top_k, s.top_p, s.min_p,
                           return_probs=c["probs"])


# ------------------------------------------------------------------------------ plain forms

def _plain_rows(s, c):
    bs = c["bs"]
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu = torch.cat([zero, s.new.clamp(min=0).cumsum(0)]).clamp(max=s.rows)
    r = torch.arange(s.rows, device=DEV)
    live = r < cu[-1]
    seq = torch.where(live, (r[:, None] >= cu[None, 1:]).sum(1), 0)
    pos = torch.where(live, s.ctx[seq] + r - cu[seq], 0)
    page = s.table[seq, pos // bs].long()
    slot = torch.where(live & (page >= 0), page * bs + pos % bs, -1)
    return (cu.to(torch.int32), torch.where(live, seq, -1).to(torch.int32),
            torch.where(live, pos, -1).to(torch.int32), slot)


def _turn(x, pos, c, f, factor, back=False):
    """x [..., heads, D] in 32 bits, its part [start, start + rot) turned by pos * f."""
    m, a = c["rot"] // 2, c["start"]
    angle = pos.double()[..., None] * f
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    cos, sin = cos[..., None, :], (-sin if back else sin)[..., None, :]
    y = x.float().clone()
    part = x[..., a:a + 2 * m].float()
    if c["pairs"]:
        u, v = part[..., 0::2], part[..., 1::2]
        y[..., a:a + 2 * m] = torch.stack((u * cos - v * sin, v * cos + u * sin), -1).flatten(-2)
    else:
        u, v = part[..., :m], part[..., m:]
        y[..., a:a + 2 * m] = torch.cat((u * cos - v * sin, v * cos + u * sin), -1)
    return y.to(x.dtype)


def _plain_append(s, c):
    rows = s.k_cache.view(-1, c["Hkv"], D), s.v_cache.view(-1, c["Hkv"], D)
    rows[0][s.slots] = _turn(s.k, s.pos, c, s.inv_freq, s.factor)
    rows[1][s.slots] = s.v
    return _turn(s.q, s.pos, c, s.inv_freq, s.factor), s.k_cache, s.v_cache


def _plain_turn(s, c):
    with torch.no_grad():
        q, k = (_turn(x, s.pos, c, s.inv_freq, s.factor) for x in (s.q, s.k))
        dq, dk = (_turn(x, s.pos, c, s.inv_freq, s.factor, back=True) for x in (s.dq, s.dk))
    return q, k, dq, dk


def _plain_shared(s, c):
    """Every request by itself over all of its keys."""
    H, Hkv, bs = c["H"], c["Hkv"], c["bs"]
    G, r0, out = H // Hkv, 0, []
    for b, (ctx, n) in enumerate(zip(*s.lens[:2])):
        S = ctx + n
        pages = s.table[b, :(S + bs - 1) // bs].long()
        k, v = (x[pages].view(-1, Hkv, D)[:S].float() for x in (s.k_cache, s.v_cache))
        q = s.q[r0:r0 + n].float().view(n, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * n, D)
        z = torch.matmul(q, k.permute(1, 2, 0).contiguous()).view(Hkv, G, n, S) * SCALE
        last = ctx + torch.arange(n, device=DEV)
        z = torch.where(torch.arange(S, device=DEV) <= last[:, None], z, -math.inf)
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(Hkv, G * n, S)
        o = torch.matmul(p, v.permute(1, 0, 2).contiguous()).view(Hkv, G, n, D)
        out.append(o.permute(2, 0, 1, 3).reshape(n, H, D))
        r0 += n
    return torch.cat(out).to(TYPES[c["out"]])


def _plain_sample(s, c):
    V = c["V"]
    x = s.logits.double()
    best = s.temperature[:, None] <= 0
    t = torch.where(best, 1.0, s.temperature[:, None].double())
    w = torch.exp((x - x.amax(-1, keepdim=True)) / t)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    place = torch.arange(V, device=DEV)[None]
    k = torch.where(best, 1, torch.where(s.top_k > 0, s.top_k, V)[:, None])
    ws = torch.where(place < k, ws, 0.0)
    mass = ws.cumsum(-1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], -1)
    keep = (before < s.top_p[:, None].double() * mass[:, -1:]) & (ws >= s.min_p[:, None].double())
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    run_ = kept.cumsum(-1)
    total = run_[:, -1:]
    token = torch.where(run_ > s.u[:, None].double() * total, place, V - 1).amin(-1)
    return (token, (kept / total).float()) if c["probs"] else token


# ------------------------------------------------------------------------------ exact

def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"rows": _exact_rows, "append": _exact_append, "turn": _exact_turn,
            "shared": _exact_shared, "sample": _exact_sample}[c["kind"]](s, c)


def _exact_rows(s, c):
    """By lists."""
    bs, table = c["bs"], s.table.tolist()
    cu, seq, pos, slot = [0], [], [], []
    for b, (ctx, n) in enumerate(zip(s.ctx.tolist(), s.new.tolist())):
        for t in range(ctx, ctx + n):
            seq.append(b)
            pos.append(t)
            slot.append(table[b][t // bs] * bs + t % bs)
        cu.append(len(seq))
    pad = [-1] * (s.rows - len(seq))
    i32 = torch.int32
    return (torch.tensor(cu, dtype=i32), torch.tensor(seq + pad, dtype=i32),
            torch.tensor(pos + pad, dtype=i32), torch.tensor(slot + pad))


def _exact_turn_of(x, pos, c, s, sign=1.0):
    """Pairs as complex numbers."""
    m, a = c["rot"] // 2, c["start"]
    x = x.detach().double()
    part = x[..., a:a + 2 * m]
    z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) if c["pairs"] \
        else torch.complex(part[..., :m].contiguous(), part[..., m:].contiguous())
    angle = sign * pos.double()[..., None, None] * s.inv_freq
    z = z * torch.polar(torch.full_like(angle, s.factor), angle)
    both = (z.real, z.imag)
    part = torch.stack(both, -1).flatten(-2) if c["pairs"] else torch.cat(both, -1)
    return torch.cat((x[..., :a], part, x[..., a + 2 * m:]), -1)


def _exact_append(s, c):
    k, v = s.k_cache.double(), s.v_cache.double()
    kr = _exact_turn_of(s.k, s.pos, c, s)
    page, at = s.slots // c["bs"], s.slots % c["bs"]
    k[page, at] = kr
    v[page, at] = s.v.double()
    return _exact_turn_of(s.q, s.pos, c, s), k, v


def _exact_turn(s, c):
    return tuple(_exact_turn_of(x, s.pos, c, s, sign)
                 for x, sign in ((s.q, 1.0), (s.k, 1.0), (s.dq, -1.0), (s.dk, -1.0)))


def _exact_shared(s, c):
    """Head by head, the prompt's keys listed from the group's first request."""
    H, Hkv, bs = c["H"], c["Hkv"], c["bs"]
    ctx, new, ways, shared = s.lens
    table, cu = s.table.cpu(), _sums(new)
    out = torch.empty(cu[-1], H, D, dtype=torch.float64, device=DEV)
    b0 = 0
    for w, p in zip(ways, shared):
        for b in range(b0, b0 + w):
            S = ctx[b] + new[b]
            at = [int(table[b0 if j < p else b, j // bs]) * bs + j % bs for j in range(S)]
            at = torch.tensor(at, device=DEV)
            for h in range(Hkv):
                k, v = (x.view(-1, Hkv, D)[at, h].double() for x in (s.k_cache, s.v_cache))
                for i in range(new[b]):
                    heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
                    m = ctx[b] + i + 1
                    z = s.q[cu[b] + i, heads].double() @ k[:m].t().contiguous() * SCALE
                    out[cu[b] + i, heads] = torch.softmax(z, -1) @ v[:m]
        b0 += w
    return out


def _exact_sample(s, c):
    """Row by row on the host."""
    R, V = c["R"], c["V"]
    tokens, probs = [], []
    x_all, u = s.logits.double().cpu().numpy(), s.u.double().tolist()
    settings = zip(s.temperature.double().tolist(), s.top_k.tolist(), s.top_p.double().tolist(),
                   s.min_p.double().tolist())
    for r, (t, k, p, m) in enumerate(settings):
        x = x_all[r]
        ids = np.lexsort((np.arange(V), -x))
        ids = ids[:1 if t <= 0 else k if k > 0 else V]
        w = np.exp((x[ids] - x[ids[0]]) / (t if t > 0 else 1.0))
        sums = np.cumsum(w)
        n = int(np.searchsorted(sums, p * sums[-1], side="left")) + 1    # the first to reach p
        keep = ids[:n][w[:n] >= m]
        full = np.zeros(V)
        full[keep] = np.exp((x[keep] - x[ids[0]]) / (t if t > 0 else 1.0))
        sums = np.cumsum(full)
        over = np.nonzero(sums > u[r] * sums[-1])[0]
        tokens.append(int(over[0]) if len(over) else int(np.nonzero(full)[0][-1]))
        probs.append(full / sums[-1])
    token = torch.tensor(tokens)
    return (token, torch.from_numpy(np.stack(probs))) if c["probs"] else token


# ------------------------------------------------------------------------------ the work

def work(case):
    c = dict(case)
    kind = c["kind"]
    if kind == "rows":
        ctx, new, _, _ = _lengths(c)
        pages = sum((n + c["bs"] - 1) // c["bs"] for n in new)
        return {"bytes": 12 * len(ctx) + 4 * pages + 16 * (sum(new) + c["spare"]),
                "flops": 4 * sum(new)}
    if kind in ("append", "turn"):
        size = 4 if c["type"] == "fp32" else 2
        tokens = c["T"] if kind == "append" else c["B"] * c["S"]
        heads = c["H"] + 2 * c["Hkv"] if kind == "append" else 2 * (c["H"] + c["Hkv"])
        turned = c["H"] + c["Hkv"] if kind == "append" else heads
        return {"bytes": tokens * (2 * heads * D * size + 12), "flops": tokens * turned * c["rot"] * 3}
    if kind == "shared":
        ctx, new, ways, shared = _lengths(c)
        own_keys, b = 0, 0
        for w, p in zip(ways, shared):
            own_keys += sum(ctx[i] + new[i] - p for i in range(b, b + w))
            b += w
        keys = sum(shared) + own_keys
        seen = sum(n * (a + (n + 1) / 2) for a, n in zip(ctx, new))
        rows = sum(new)
        out = 2 if c["out"] == "bf16" else 4
        return {"bytes": keys * c["Hkv"] * D * 4 + rows * c["H"] * D * (2 + out),
                "flops": 4.0 * seen * c["H"] * D}
    size = 4 if c["type"] == "fp32" else 2
    return {"bytes": c["R"] * c["V"] * (size + (4 if c["probs"] else 0)) + 32 * c["R"],
            "flops": 4.0 * c["R"] * c["V"]}
