"""Trees of drafted tokens in plain Python and 64 bits: their attention, their verification and
the pages of a cache, one row, node or page at a time."""

import math

import torch


def ancestors(parents, i):
    """Node i and its ancestors, deepest first."""
    out = []
    while i >= 0:
        out.append(i)
        p = parents[i]
        i = p if 0 <= p < i else -1
    return out


def attend(q, k, v, idx, bias, valid, seen, depth, ctx, bs, lw, scale):
    """Rows q [n,H,D] of one sequence over its keys k, v [S,Hkv,D]: seen[i] the drafted nodes that
    row i sees, depth[i]; idx, bias, valid [n,K] or None.  (out [n,H,D], lse [n,H]) in 64 bits."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64)
    for i in range(n):
        w = ctx + int(depth[i]) - lw + 1
        keys, extra, done = list(range(max(w, 0), ctx)), [0.0] * (ctx - min(max(w, 0), ctx)), set()
        keys += [ctx + m for m in seen[i]]
        extra += [0.0] * len(seen[i])
        for s in range(0 if idx is None else idx.shape[1]):
            c = int(idx[i, s])
            if c < 0 or c in done or (valid is not None and not bool(valid[i, s])):
                continue
            block = range(c * bs, min((c + 1) * bs, w, ctx))
            if len(block):
                done.add(c)
                keys += list(block)
                extra += [float(bias[i, s])] * len(block)
        if not keys:
            continue
        for h in range(H):
            z = k[keys, h // G].double() @ q[i, h].double() * scale
            z = z + torch.tensor(extra, dtype=torch.float64)
            lse[i, h] = torch.logsumexp(z, 0)
            out[i, h] = torch.softmax(z, 0) @ v[keys, h // G].double()
    return out, lse


def verify(target, tokens, parents, u=None, draft=None):
    """(path, next token) of one sequence: target [n,V], tokens, parents lists."""
    n = target.shape[0]
    if n == 0:
        return [], -1
    at, path = 0, [0]
    while True:
        kids = [i for i in range(at + 1, n) if parents[i] == at]
        if u is None:
            row = target[at].float()
            row = torch.where(row.isnan(), -math.inf, row)
            best = int((row == row.max()).nonzero()[0])
            hit = [i for i in kids if tokens[i] == best]
            if not hit:
                return path, best
            at = hit[0]
            path.append(at)
            continue
        row = torch.where(target[at].double() > 0, target[at].double(), 0.0)
        q = None if draft is None else torch.where(draft[at].double() > 0, draft[at].double(), 0.0)
        rest, mass, found = row.clone(), 1.0, None
        for i in kids:
            x = tokens[i]
            inside = 0 <= x < row.numel()
            share = 1.0 if q is None or not inside else float(q[x])
            have = float(rest[x]) if inside else 0.0
            if float(u[i]) * mass * share < have:
                found = i
                break
            if q is not None:
                rest = (rest - mass * q).clamp(min=0)
                mass = float(rest.sum())
            elif inside:
                mass -= have
                rest[x] = 0.0
        if found is not None:
            at = found
            path.append(at)
            continue
        rest = rest if float(rest.sum()) > 0 else row
        if not float(rest.sum()) > 0:
            return path, -1
        run = rest.cumsum(0)
        over = (run > float(u[0]) * float(run[-1])).nonzero()
        return path, int(over[0]) if len(over) else int((rest > 0).nonzero()[-1])


class Pages:
    """refs, table and lens as lists; the moves of the last call in `moves`."""

    def __init__(self, num_pages, rows, width, page):
        self.refs = [0] * num_pages
        self.table = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.page = page

    def blocks(self, n):
        return -(-n // self.page)

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def fork(self, src, dst):
        tails = sum(self.lens[s] % self.page > 0 for s in src)
        if len(set(dst)) < len(dst) or any(self.lens[d] for d in dst) or set(src) & set(dst) \
                or tails > self.refs.count(0):
            return 0, [-1] * len(src), [-1] * len(src)
        frm, to = [], []
        for s, d in zip(src, dst):
            n = self.lens[s]
            for i in range(n // self.page):
                self.table[d][i] = self.table[s][i]
                self.refs[self.table[s][i]] += 1
            frm.append(-1)
            to.append(-1)
            if n % self.page:
                i = n // self.page
                frm[-1] = self.table[s][i]
                to[-1] = self.table[d][i] = self._take()
            self.lens[d] = n
        return 1, frm, to

    def reserve(self, new):
        R = len(self.lens)
        need, shared = 0, [False] * R
        for r, n in enumerate(new):
            if n <= self.lens[r]:
                continue
            if n > len(self.table[r]) * self.page:
                return 0, [-1] * R, [-1] * R
            tail = self.lens[r] % self.page
            shared[r] = tail > 0 and self.refs[self.table[r][self.lens[r] // self.page]] > 1
            need += self.blocks(n) - self.blocks(self.lens[r]) + shared[r]
        if need > self.refs.count(0):
            return 0, [-1] * R, [-1] * R
        frm, to = [-1] * R, [-1] * R
        for r, n in enumerate(new):
            if n <= self.lens[r]:
                continue
            if shared[r]:
                i = self.lens[r] // self.page
                frm[r] = self.table[r][i]
                to[r] = self.table[r][i] = self._take()
            for i in range(self.blocks(self.lens[r]), self.blocks(n)):
                self.table[r][i] = self._take()
            self.lens[r] = n
        for p in frm:
            if p >= 0:
                self.refs[p] -= 1
        return 1, frm, to

    def free(self, keep):
        for r, n in enumerate(keep):
            n = max(n, 0)
            for i in range(self.blocks(n), self.blocks(self.lens[r])):
                self.refs[self.table[r][i]] -= 1
                self.table[r][i] = -1
            self.lens[r] = min(n, self.lens[r])

    def compact(self):
        live = sum(x > 0 for x in self.refs)
        frm = [p for p in range(live, len(self.refs)) if self.refs[p]]
        to = [p for p in range(live) if not self.refs[p]]
        place = dict(zip(frm, to))
        for a, b in place.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[place.get(p, p) if i < self.blocks(n) else -1 for i, p in enumerate(row)]
                      for row, n in zip(self.table, self.lens)]
        return frm, to
