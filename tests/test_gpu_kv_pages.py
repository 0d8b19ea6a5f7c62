"""Pages of a cache (kv_pages) against lists: tables, counts and contents have to be equal."""

import pytest
import torch

from ananta_ocr_amd import kv_pages
from tree_oracle import Pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _pool(num_pages=24, rows=6, width=7, page=8, layers=2):
    k = torch.zeros(layers, num_pages, page, 3, 16, dtype=torch.bfloat16, device=DEV)
    ik = torch.zeros(layers, num_pages, page, 12, device=DEV)
    kb = torch.zeros(layers, num_pages, 12, device=DEV)
    caches = kv_pages.PageCaches([k, ik], pages=[kb], layered=True)
    return kv_pages.PagePool(caches, rows, width), (k, ik, kb), Pages(num_pages, rows, width, page)


def _same(pool, lists):
    assert pool.refs.tolist() == lists.refs
    assert pool.lens.tolist() == lists.lens
    assert pool.table.tolist() == lists.table


class Shadow:
    """What every row should read: a number per token (and per page, of its first token)."""

    def __init__(self, pool, tensors, lists):
        self.pool, self.t, self.lists = pool, tensors, lists
        self.rows = [[] for _ in lists.lens]
        self.n = 0

    def write(self, r, start):
        """Numbers of the row's tokens from `start` on into the caches, through the table."""
        page = self.lists.page
        for j in range(start, self.lists.lens[r]):
            self.n += 1
            self.rows[r][j:] = [self.n % 251]
            p = self.lists.table[r][j // page]
            for t in self.t[:2]:
                t[:, p, j % page] = self.n % 251
            self.t[2][:, p] = self.rows[r][j // page * page]

    def check(self):
        page = self.lists.page
        for r, row in enumerate(self.rows):
            assert len(row) == self.lists.lens[r]
            for t in self.t[:2]:
                if row:
                    pages = torch.tensor(self.lists.table[r][:-(-len(row) // page)], device=DEV)
                    got = t[:, pages].flatten(3).flatten(1, 2)[:, :len(row)]
                    want = torch.tensor(row, device=DEV, dtype=t.dtype)[None, :, None]
                    assert torch.equal(got, want.expand_as(got)), r


@pytest.mark.parametrize("seed", range(4))
def test_a_pool_through_many_steps(seed):
    """Rows reserved, forked, written, cut and compacted in any order, with the pool running
    short: state equal to the lists', every row's content what was written to it."""
    g = torch.Generator().manual_seed(seed)

    def rnd(n):
        return int(torch.randint(0, n, (1,), generator=g))
    pool, tensors, lists = _pool()
    sh = Shadow(pool, tensors, lists)
    refused = 0
    for _ in range(60):
        what = rnd(5)
        if what <= 1:
            new = [n + rnd(13) if rnd(2) else rnd(9) for n in lists.lens]
            if rnd(8) == 0:
                new[rnd(6)] = 57                               # past the table's width
            old = list(lists.lens)
            ok = pool.reserve(_i32(new))
            want, _, _ = lists.reserve(new)
            assert int(ok) == want
            refused += not want
            for r, n in enumerate(old):
                if want and new[r] > n:
                    sh.write(r, n)
        elif what == 2:
            src = [rnd(6) for _ in range(1 + rnd(3))]
            dst = [rnd(6) for _ in src]
            ok = pool.fork(_i32(src), _i32(dst))
            want, _, _ = lists.fork(src, dst)
            assert int(ok) == want
            if want:
                for a, b in zip(src, dst):
                    sh.rows[b] = list(sh.rows[a])
        elif what == 3:
            keep = [rnd(n + 1) if rnd(3) == 0 else (0 if rnd(4) == 0 else n + rnd(3))
                    for n in lists.lens]
            keep[rnd(6)] -= 100 * (rnd(6) == 0)
            pool.free(_i32(keep))
            lists.free(keep)
            for r, n in enumerate(keep):
                del sh.rows[r][max(n, 0):]
        else:
            pool.compact()
            lists.compact()
        _same(pool, lists)
        sh.check()
        counts = [0] * 24
        for row in lists.table:
            for p in row:
                if p >= 0:
                    counts[p] += 1
        assert counts == lists.refs
    assert refused


def test_large_pools_and_tables():
    """More pages, rows and pairs than a work-group has lanes."""
    for num_pages, rows, width, page in ((5000, 1500, 3, 16), (2049, 3, 1024, 1)):
        g = torch.Generator().manual_seed(num_pages)
        k = torch.randn(num_pages, page, 4, device=DEV)
        pool = kv_pages.PagePool(kv_pages.PageCaches([k]), rows, width)
        lists = Pages(num_pages, rows, width, page)
        half = rows // 2 + 1
        new = [int(x) if r < half else 0 for r, x in
               enumerate(torch.randint(1, width * page + 1, (rows,), generator=g))]
        assert int(pool.reserve(_i32(new))) == lists.reserve(new)[0]
        _same(pool, lists)
        src = list(range(rows - half))
        dst = list(range(half, rows))
        old = k.clone()
        ok, frm, to = kv_pages.fork_pages(pool.refs, pool.table, pool.lens, _i32(src), _i32(dst), page)
        want = lists.fork(src, dst)
        assert (int(ok), frm.tolist(), to.tolist()) == want
        kv_pages.copy_pages(pool.caches, frm, to)
        f, t = (torch.tensor([p for p in x if p >= 0], dtype=torch.long, device=DEV) for x in want[1:])
        old[t] = old[f]
        assert torch.equal(k, old)
        keep = [int(x) for x in torch.randint(0, width * page, (rows,), generator=g)]
        keep[::3] = [0] * len(keep[::3])
        pool.free(_i32(keep))
        lists.free(keep)
        _same(pool, lists)
        refs, table, frm, to = kv_pages.compact_pages(pool.refs, pool.table, pool.lens, page)
        _same(pool, lists)                                     # the given state stays
        f, t = lists.compact()
        pad = [-1] * (num_pages // 2 - len(f))
        assert frm.tolist() == f + pad and to.tolist() == t + pad
        assert refs.tolist() == lists.refs and table.tolist() == lists.table


def test_refused_forks_change_nothing():
    pool, _, lists = _pool()
    for n in ([13, 8, 0, 0, 0, 0],):
        pool.reserve(_i32(n))
        lists.reserve(n)
    for src, dst in (([0], [1]), ([0, 0], [2, 2]), ([0, 2], [2, 3]), ([6], [2]), ([0], [6]),
                     ([-1], [2]), ([0], [-1])):
        ok, frm, to = kv_pages.fork_pages(pool.refs, pool.table, pool.lens, _i32(src), _i32(dst), 8)
        assert int(ok) == 0 and frm.tolist() == to.tolist() == [-1] * len(src)
        _same(pool, lists)
    # a table entry that is no page
    pool.table[0, 1] = 10 ** 6
    ok, _, _ = kv_pages.fork_pages(pool.refs, pool.table, pool.lens, _i32([0]), _i32([3]), 8)
    assert int(ok) == 0 and pool.lens.tolist() == lists.lens and pool.refs.tolist() == lists.refs
    ok, _, _ = kv_pages.reserve_pages(pool.refs, pool.table, pool.lens, _i32([14] + [0] * 5), 8)
    assert int(ok) == 0 and pool.lens.tolist() == lists.lens and pool.refs.tolist() == lists.refs
    # no pairs, no pages to hand out
    ok, frm, to = kv_pages.fork_pages(pool.refs, pool.table, pool.lens, _i32([]), _i32([]), 8)
    assert int(ok) == 1 and frm.numel() == 0
    kv_pages.copy_pages(pool.caches, frm, to)
    pool.refs.fill_(1)
    ok, _, _ = kv_pages.reserve_pages(pool.refs, pool.table, pool.lens, _i32([13, 9, 0, 0, 0, 0]), 8)
    assert int(ok) == 0 and pool.lens.tolist() == lists.lens


def test_lengths_that_are_none():
    """A length past the table is refused, one past any sum of 32 bits too."""
    for length in (2 ** 31 - 1, 2 ** 31 - 8, 10 ** 9, -1):
        pool, _, _ = _pool()
        pool.lens[0] = length
        for f, rows in ((kv_pages.fork_pages, (_i32([0]), _i32([3]))),
                        (kv_pages.reserve_pages, (_i32([1] * 6),))):
            before = pool.table.clone(), pool.refs.clone(), pool.lens.clone()
            ok, frm, to = f(pool.refs, pool.table, pool.lens, *rows, 8)
            assert int(ok) == 0 and frm.tolist() == to.tolist() == [-1] * frm.numel()
            assert all(torch.equal(x, y) for x, y in zip(before, (pool.table, pool.refs, pool.lens)))


@pytest.mark.parametrize("dtype,inner", [
    (torch.bfloat16, (10, 128)), (torch.float32, (128,)), (torch.float32, (3,)),
    (torch.bfloat16, (5, 7)), (torch.int8, (9,)), (torch.float16, (1, 3)), (torch.float64, ()),
    (torch.uint8, (4096,))])
def test_copies_of_every_unit(dtype, inner):
    """Pages of every element size; pairs that name no page are left out."""
    x = torch.randint(0, 200, (3, 19, 6, *inner), device=DEV).to(dtype)
    want = x.clone()
    frm, to = [4, -1, 0, 18, 19, 2, 10 ** 9], [7, 3, -1, 1, 5, 40, 6]
    want[:, [7, 1]] = want[:, [4, 18]]
    kv_pages.copy_pages(kv_pages.PageCaches([x], layered=True), _i32(frm), _i32(to))
    assert torch.equal(x, want)


def test_copies_of_pages_of_one_token():
    """An axis of one token, of any stride, and more caches than one launch takes."""
    base = torch.arange(40 * 9 * 16, dtype=torch.float32, device=DEV).view(40, 1, 9, 16)
    keep = base.clone()
    views = [base[i].transpose(0, 1) for i in range(40)]         # [9, 1, 16], strides (16, 144, 1)
    assert views[0].stride() == (16, 144, 1) and views[0].is_contiguous()
    caches = kv_pages.PageCaches(views)
    kv_pages.copy_pages(caches, _i32([2, 8]), _i32([5, 0]))
    keep[:, 0, 5], keep[:, 0, 0] = keep[:, 0, 2].clone(), keep[:, 0, 8].clone()
    assert torch.equal(base, keep)


def test_copies_of_strided_caches():
    """Keys and values of one interleaved pool, heads outside the tokens, a view that leaves
    columns out (which stay), more caches than a launch takes."""
    base = torch.randn(11, 2, 6, 4, 32, device=DEV).bfloat16()
    want = base.clone()
    want[5] = want[2]
    kv_pages.copy_pages(kv_pages.PageCaches([base[:, 0], base[:, 1]]), _i32([2]), _i32([5]))
    assert torch.equal(base, want)
    heads = torch.randn(11, 4, 6, 32, device=DEV)
    want = heads.clone()
    want[5] = want[2]
    kv_pages.copy_pages(kv_pages.PageCaches([heads.transpose(1, 2)]), _i32([2]), _i32([5]))
    assert torch.equal(heads, want)
    wide = torch.randn(11, 6, 4, 40, device=DEV)
    want = wide.clone()
    want[5, :, :, 3:35] = want[2, :, :, 3:35]
    kv_pages.copy_pages(kv_pages.PageCaches([wide[..., 3:35]]), _i32([2]), _i32([5]))
    assert torch.equal(wide, want)
    many = [torch.randn(7, 4, 1 + i, device=DEV) for i in range(70)]
    want = [t.clone() for t in many]
    for t in want:
        t[6], t[3] = t[1].clone(), t[0].clone()
    kv_pages.copy_pages(kv_pages.PageCaches(many), _i32([1, 0]), _i32([6, 3]))
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    with pytest.raises(NotImplementedError):
        kv_pages.PageCaches([torch.zeros(4, 6, 8, 8, 8, device=DEV)[:, ::2, ::2, ::2]])
    with pytest.raises(ValueError):
        kv_pages.PageCaches([torch.zeros(4, 1, 8, device=DEV).expand(4, 6, 8)])


def _keep_ref(tensors, path, count, ctx, table, page, layered):
    for b, (p, m) in enumerate(zip(path, count)):
        for t in tensors:
            at = (slice(None),) if layered else ()
            rows = [t[at + (table[b][(ctx[b] + x) // page], (ctx[b] + x) % page)].clone()
                    for x in p[:m]]
            for i, r in enumerate(rows):
                j = ctx[b] + i
                t[at + (table[b][j // page], j % page)] = r


@pytest.mark.parametrize("page,shape,dtype", [(8, (3, 16), torch.bfloat16), (64, (10, 128), torch.bfloat16),
                                              (5, (7,), torch.float32), (4, (3,), torch.int8)])
def test_accepted_rows(page, shape, dtype):
    """Paths whose sources are places that other rows move to, long ones, ones that stay, across
    pages; the caches of every layer, and nothing else."""
    g = torch.Generator().manual_seed(page)
    nodes = [1, 12, 100, 200, 30, 5]
    ctx = [0, page - 1, 3 * page, 7, page * 2 - 3, 1]
    path, count = [], []
    for n in nodes:
        m = 1 + int(torch.randint(0, n, (1,), generator=g))
        rest = (torch.randperm(n - 1, generator=g)[:m - 1] + 1).sort().values.tolist()
        path.append([0] + rest + [-1] * (200 - m))
        count.append(m)
    path[5], count[5] = [-1] * 200, 0                          # a request without nodes
    path[4] = list(range(30)) + [-1] * 170
    count[4] = 30
    need = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
    perm = torch.randperm(sum(need), generator=g).tolist()
    table = [[perm.pop() if i < m else -1 for i in range(max(need))] for m in need]
    x = torch.randint(0, 100, (2, sum(need), page, *shape)).to(dtype).to(DEV)
    y = torch.randint(0, 100, (2, sum(need), page, 12)).float().to(DEV)
    want = [x.clone(), y.clone()]
    _keep_ref(want, path, count, ctx, table, page, True)
    kv_pages.keep_rows(kv_pages.PageCaches([x, y], layered=True), _i32(path), _i32(count), _i32(ctx),
                       _i32(table))
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_rows_outside_the_table_stay():
    """Entries that name no page, slots past the table, lengths below 0: left out."""
    x = torch.randn(6, 4, 8, device=DEV)
    want = x.clone()
    caches = kv_pages.PageCaches([x])
    table = _i32([[0, 1], [10 ** 8, -3], [2, 3], [4, 5]])
    path = _i32([[0, 2, 40]] * 2 + [[0, 2, 3]] * 2)
    kv_pages.keep_rows(caches, path, _i32([3, 3, 3, -2]), _i32([3, 0, -9, 0]), table)
    want[1, 0] = want[1, 1]
    assert torch.equal(x, want)


def test_a_contiguous_cache_is_a_page_a_sequence():
    x = torch.randn(3, 2, 50, 16, device=DEV)                  # [B, H, S, D]
    want = x.clone()
    for b, c in enumerate((10, 0, 44)):
        want[b, :, c + 1] = x[b, :, c + 3]
        want[b, :, c + 2] = x[b, :, c + 4]
    kv_pages.keep_rows(kv_pages.PageCaches([x.transpose(1, 2)]), _i32([[0, 3, 4]] * 3), _i32([3] * 3),
                       _i32([10, 0, 44]), _i32([[0], [1], [2]]))
    assert torch.equal(x, want)


def test_offsets_past_32_bits():
    x = torch.empty(9000, 64, 8192, dtype=torch.uint8, device=DEV)      # 4.7e9 bytes
    x[:4] = torch.randint(0, 255, (4, 64, 8192), device=DEV, dtype=torch.uint8)
    caches = kv_pages.PageCaches([x])
    kv_pages.copy_pages(caches, _i32([0, 3]), _i32([8999, 8500]))
    assert torch.equal(x[8999], x[0]) and torch.equal(x[8500], x[3])
    row = x[8999, 9].clone()
    kv_pages.keep_rows(caches, _i32([[0, 5]]), _i32([2]), _i32([4]), _i32([[8999]]))
    assert torch.equal(x[8999, 5], row)


def test_graphs_and_streams():
    """A step's page calls recorded once and replayed: the state the eager calls give."""
    pool, tensors, lists = _pool()
    eager, etensors, _ = _pool()
    for t, u in zip(tensors, etensors):
        t.copy_(torch.randint(0, 99, t.shape, device=DEV))
        u.copy_(t)
    new = torch.zeros(6, dtype=torch.int32, device=DEV)
    keep = torch.zeros(6, dtype=torch.int32, device=DEV)
    src, dst = _i32([0, 1]), _i32([4, 5])

    def step(p):
        a = p.reserve(new)
        b = p.fork(src, dst)
        p.free(keep)
        p.compact()
        return a, b
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pool)
    for i in range(5):
        new.copy_(_i32([9 + 4 * i, 16, 3 * i, 0, 0, 0]))
        keep.copy_(_i32([9 + 4 * i, 11, i, 0, 5 if i == 4 else 0, 0]))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            got = step(eager)
        torch.cuda.synchronize()
        assert [int(x) for x in out] == [int(x) for x in got]
        for x in ("refs", "table", "lens"):
            assert torch.equal(getattr(pool, x), getattr(eager, x))
        for t, u in zip(tensors, etensors):
            assert torch.equal(t, u)
