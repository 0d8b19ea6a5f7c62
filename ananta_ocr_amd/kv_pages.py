"""Pages of a paged cache on the HIP kernels (csrc/dash_kvpages.hip): copied, shared between
sequences (fork), handed out (reserve), given back (free) and moved together (compact), the rows of
accepted drafted tokens moved up (keep), and the slots of a step's new tokens (step_rows).

The state is three int32 tensors on the GPU: ``refs`` [num_pages], how many table entries name a
page (0: free); ``table`` [R, P], the pages of every sequence row; ``lens`` [R], the tokens of a
row, whose first ceil(lens / page_size) entries are in use.  Free pages are handed out lowest
first, to the rows in order.  Nothing synchronises: calls that can fail return ``ok`` (int32 [1]
on the GPU; where it is 0 nothing was changed).

The outputs of a call are views of one allocation (some KB); clone what is kept for long or saved.

``PagePool`` holds the state and the caches and keeps them consistent; the functions are its
parts.  ``PageCaches`` describes the tensors that the pages lie in, once for many calls.
"""

import ctypes
import functools
import math

import torch

from . import _lib
from .ops import _i32, _ptr, _stream
from .tree import _device, _shape

MAX_ROWS = 8192
MAX_STEP_TOKENS = 2 ** 31 - 2       # of a table row, that a step's refusal must pass


class PageCaches:
    """The tensors that hold a pool's pages: ``tokens`` of [num_pages, page_size, ...] each (keys,
    values, index keys: a row per token) and ``pages`` of [num_pages, ...] (block summaries: a
    row per page); with ``layered`` every tensor has a leading layer axis.  Any types and strides
    whose innermost piece is contiguous and that do not overlap; every tensor on one GPU and of the
    same number of pages.  Addresses are noted once: the tensors keep their memory (no resize_ or
    set_) while the object is in use."""

    def __init__(self, tokens, pages=(), layered=False):
        self.tensors = [*tokens, *pages]
        if not self.tensors:
            raise ValueError("a pool needs at least one cache")
        if not tokens:
            raise ValueError("a pool needs a cache with a row per token")
        ax = 1 if layered else 0
        _device(*self.tensors)
        first = self.tensors[0]
        self.device = first.device
        if first.dim() < ax + 2:
            raise ValueError("a cache of [num_pages, page_size, ...] is needed")
        self.num_pages, self.page_size = first.shape[ax:ax + 2]
        head = (self.num_pages, self.page_size)
        if 0 in head:
            raise ValueError(f"caches of {head} pages and tokens")
        for i, t in enumerate(self.tensors):
            if t.requires_grad:
                raise ValueError("a cache that requires grad cannot be written in place")
            n = 2 if i < len(tokens) else 1
            if t.shape[ax:ax + n] != head[:n]:
                raise ValueError(f"caches of {head} pages and tokens, and of shape {tuple(t.shape)}")
        self._ax, self._tokens = ax, len(tokens)
        if not all(t.is_contiguous() for t in self.tensors):
            self._copy, self._rows           # refuse layouts here

    @functools.cached_property
    def _copy(self):
        return self._describe([(t, self._ax + 1) for t in self.tensors if t.numel()], self._ax)

    @functools.cached_property
    def _rows(self):
        return self._describe([(t, self._ax + 2) for t in self.tensors[:self._tokens] if t.numel()],
                              self._ax)

    @staticmethod
    def _describe(tensors, ax):
        """(count, addresses, descriptors) as the C entry points take them: the axes from `at` on
        are joined where they lie in one piece."""
        n = len(tensors)
        base, desc = [], []
        for t, at in tensors:
            size, stride, es = t.shape, t.stride(), t.element_size()
            rows = at == ax + 2
            if t.is_contiguous():            # a page, or a row, in one piece
                base.append(t.data_ptr())
                seg = es * math.prod(size[at:])    # (an axis of one may have any stride)
                desc += (size[0] if ax else 1, stride[0] * es if ax else 0, stride[ax] * es, 1,
                         stride[ax + 1] * es if rows else 0, 1, 0, seg)
                continue
            seg, dims = 1, []                # by stride: source and target share the order
            for a in sorted(range(at, t.dim()), key=lambda a: stride[a]):
                if size[a] == 1:
                    continue
                if not dims and stride[a] == seg:
                    seg *= size[a]
                elif dims and stride[a] == dims[-1][0] * dims[-1][1]:
                    dims[-1] = (dims[-1][0] * size[a], dims[-1][1])
                else:
                    dims.append((size[a], stride[a]))
            reach = seg
            for count, st in dims:
                if st < reach:
                    raise ValueError("a cache with overlapping rows")
                reach = st * (count - 1) + reach
            for a in range(at):
                if size[a] > 1 and stride[a] <= 0:
                    raise ValueError("a cache with overlapping pages")
            if len(dims) > (1 if rows else 2):
                raise NotImplementedError(
                    f"cache of shape {tuple(size)} and strides {tuple(stride)}: its pages lie in "
                    "pieces of more than two levels")
            dims += [(1, 0)] * (2 - len(dims))
            (n2, s2), (n1, s1) = dims[0], dims[1]
            if rows:
                n1, s1 = 1, stride[ax + 1]
            base.append(t.data_ptr())
            desc += (size[0] if ax else 1, stride[0] * es if ax else 0, stride[ax] * es, n1,
                     s1 * es, n2, s2 * es, seg * es)
        return n, (ctypes.c_void_p * max(n, 1))(*base), (ctypes.c_int64 * max(8 * n, 1))(*desc)


def copy_pages(caches, from_pages, to_pages):
    """The content of page from_pages[i] to page to_pages[i] in every cache (PageCaches); pairs
    with a number that names no page (-1) are left out.  No page may be both a source and a
    target, or the target of two pairs."""
    _shape(to_pages, from_pages.shape, "to_pages")
    with _device(caches.tensors[0], from_pages, to_pages):
        f, t = _i32(from_pages), _i32(to_pages)
        n, base, desc = caches._copy
        _lib.check(_lib.load().dash_copy_pages(n, base, desc, _ptr(f), _ptr(t), f.numel(),
                                               caches.num_pages, _stream()), "dash_copy_pages")


def keep_rows(caches, path, count, context_lens, table):
    """The rows of accepted nodes moved up in every cache with a row per token: slot
    context_lens[b] + path[b, i] -> context_lens[b] + i, 1 <= i < count[b], as tree.verify_tree
    gives path [B, n] and count [B] (path is strictly increasing).  table [B, P]."""
    B, n = path.shape
    for x, what in ((count, "count"), (context_lens, "context_lens")):
        _shape(x, (B,), what)
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table: {B} rows needed")
    with _device(caches.tensors[0], path, count, context_lens, table):
        p, c, ctx, bt = (_i32(x) for x in (path, count, context_lens, table))
        m, base, desc = caches._rows
        _lib.check(_lib.load().dash_keep_rows(
            m, base, desc, _ptr(p), n, _ptr(c), _ptr(ctx), _ptr(bt), bt.stride(0), B, bt.shape[1],
            caches.page_size, caches.num_pages, n, _stream()), "dash_keep_rows")


def _keep_lens(path, count, context_lens, lens):
    """(stand, kept, new_context, summed) of a verified step's rows, int32 [B] each
    (dash_keep_lens)."""
    B, n = path.shape
    for x, what in ((count, "count"), (context_lens, "context_lens"), (lens, "lens")):
        _shape(x, (B,), what)
    with _device(lens, path, count, context_lens):
        p, c, ctx, ln = (_i32(x) for x in (path, count, context_lens, lens))
        out = _ints(lens.device, B, B, B, B)
        _lib.check(_lib.load().dash_keep_lens(_ptr(p), n, _ptr(c), _ptr(ctx), _ptr(ln), B, n,
                                              *(_ptr(x) for x in out), _stream()), "dash_keep_lens")
    return out


def _state(refs, table, lens, page_size):
    if refs.dim() != 1 or refs.numel() == 0 or table.dim() != 2:
        raise ValueError("refs [num_pages] and table [R, P] are needed")
    _shape(lens, (table.shape[0],), "lens")
    if table.shape[0] > MAX_ROWS:
        raise NotImplementedError(f"tables of at most {MAX_ROWS} rows")
    if int(page_size) < 1:
        raise ValueError(f"page_size {page_size}")


def _in_place(**ts):
    """Tensors that a call writes: int32, with contiguous rows that do not overlap."""
    for name, t in ts.items():
        if t.dtype != torch.int32 or (t.shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name}: contiguous int32 rows are needed (written in place)")
        if t.dim() > 1 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
            raise ValueError(f"{name}: rows that overlap (written in place)")


def _ints(device, *sizes):
    """int32 tensors of one allocation (an allocation costs the host 1.3 us, a view of it 0.4)."""
    return torch.empty(sum(sizes), dtype=torch.int32, device=device).split_with_sizes(sizes)


def step_rows(table, context_lens, query_lens, page_size, num_pages, rows, lens=None):
    """Where the new tokens of a step go: request b brings query_lens[b] of them (a number below 0
    counts as 0) after its context_lens[b], packed in order into a batch of `rows` rows.  Returns
    (cu_seqlens_q int32 [B + 1], seq int32 [rows], positions int32 [rows], slots int64 [rows]): the
    prefix sums, cut to the rows, and every row's request, position (context + its place among the
    new ones) and slot in the pool, table[seq, position // page_size] * page_size + position %
    page_size.  Rows of no request hold -1, and a row's slot is -1 where the table [B, P] has no page
    for it (an entry that is none of num_pages) or, with lens [B] given, where its position is not
    below lens: after a reserve_pages that was refused a last page may be another row's too.
    At most 8,192 requests."""
    if table.dim() != 2:
        raise ValueError("table [B, P] is needed")
    B, P = table.shape
    for x, what in ((context_lens, "context_lens"), (query_lens, "query_lens"), (lens, "lens")):
        _shape(x, (B,), what)
    rows = int(rows)
    if int(page_size) < 1 or int(num_pages) < 0 or not 0 <= rows < 2 ** 31:
        raise ValueError(f"page_size {page_size}, {num_pages} pages, {rows} rows")
    if B > MAX_ROWS:
        raise NotImplementedError(f"tables of at most {MAX_ROWS} rows")
    with _device(table, context_lens, query_lens, lens):
        bt, ctx, n, ln = _i32(table), _i32(context_lens), _i32(query_lens), _i32(lens)
        slots, cu, seq, pos = _ints(bt.device, 2 * rows, B + 1, rows, rows)
        _lib.check(_lib.load().dash_step_rows(
            _ptr(n), _ptr(ctx), _ptr(ln), _ptr(bt), bt.stride(0), B, P, int(page_size),
            int(num_pages), rows, _ptr(cu), _ptr(seq), _ptr(pos), _ptr(slots), _stream()),
            "dash_step_rows")
    return cu, seq, pos, slots.view(torch.int64)


def fork_pages(refs, table, lens, src, dst, page_size):
    """Row dst[i], which is empty, becomes row src[i]: its filled pages are shared, a partly filled
    last one gets a page of its own.  refs, table and lens in place.  Returns (ok, from_pages,
    to_pages) with the pages to copy (copy_pages; -1: none).  ok is 0, and nothing changed, where
    a row is out of range, a target is filled, repeated or a source, or pages do not suffice."""
    _state(refs, table, lens, page_size)
    _in_place(refs=refs, table=table, lens=lens)
    _shape(dst, src.shape, "dst")
    n = src.numel()
    if n > MAX_ROWS:
        raise NotImplementedError(f"at most {MAX_ROWS} forks a call")
    with _device(refs, table, lens, src, dst):
        s, d = _i32(src), _i32(dst)
        ok, frm, to = _ints(refs.device, 1, n, n)
        R, P = table.shape
        _lib.check(_lib.load().dash_fork_pages(
            _ptr(refs), refs.numel(), _ptr(table), table.stride(0), R, P, _ptr(lens), _ptr(s),
            _ptr(d), n, int(page_size), _ptr(ok), _ptr(frm), _ptr(to), _stream()),
            "dash_fork_pages")
    return ok, frm, to


def reserve_pages(refs, table, lens, new_lens, page_size):
    """Rows grow to new_lens [R] tokens (shorter ones stay): pages for the blocks they lack, and a
    page of its own for the partly filled last page of a growing row that another row shares.
    refs, table and lens in place.  Returns (ok, from_pages [R], to_pages [R]) with the pages to
    copy.  ok is 0, and nothing changed, where a length does not fit the table or pages do not
    suffice; the new tokens then have no pages of their own to be written to.  Tables of at most
    2^31 - 1 entries."""
    _state(refs, table, lens, page_size)
    _in_place(refs=refs, table=table, lens=lens)
    _shape(new_lens, lens.shape, "new_lens")
    with _device(refs, table, lens, new_lens):
        nl = _i32(new_lens)
        R, P = table.shape
        ok, frm, to = _ints(refs.device, 1, R, R)
        if R == 0:
            return ok.fill_(1), frm, to
        _lib.check(_lib.load().dash_reserve_pages(
            _ptr(refs), refs.numel(), _ptr(table), table.stride(0), R, P, _ptr(lens), _ptr(nl),
            int(page_size), _ptr(ok), _ptr(frm), _ptr(to), _stream()), "dash_reserve_pages")
    return ok, frm, to


def free_pages(refs, table, lens, keep_lens, page_size):
    """Rows longer than keep_lens [R] are cut to it (0: the row leaves); the table entries above
    come out as -1 and their pages lose a name.  refs, table and lens in place."""
    _state(refs, table, lens, page_size)
    _in_place(refs=refs, table=table, lens=lens)
    _shape(keep_lens, lens.shape, "keep_lens")
    with _device(refs, table, lens, keep_lens):
        kl = _i32(keep_lens)
        R, P = table.shape
        if R and P:
            _lib.check(_lib.load().dash_free_pages(
                _ptr(refs), refs.numel(), _ptr(table), table.stride(0), R, P, _ptr(lens), _ptr(kl),
                int(page_size), _stream()), "dash_free_pages")


def compact_pages(refs, table, lens, page_size):
    """The pages in use moved to the lowest numbers: with L of them, the i-th at or above L goes to
    the i-th free page below it.  Returns (refs, table, from_pages, to_pages): the state after the
    moves (table entries not in use: -1) and the pages to copy, [num_pages / 2] and -1 past them.
    The given state stays as it is, for launches that still read it."""
    _state(refs, table, lens, page_size)
    with _device(refs, table, lens):
        r, t, ln = _i32(refs), _i32(table), _i32(lens)
        n = r.numel()
        R, P = t.shape
        moves = max(n // 2, 1)
        new_refs, new_table, frm, to, place = _ints(r.device, n, R * P, moves, moves, n)
        new_table = new_table.view(R, P)
        _lib.check(_lib.load().dash_compact_pages(
            _ptr(r), n, _ptr(t), t.stride(0), R, P, _ptr(ln), int(page_size), _ptr(new_refs),
            _ptr(new_table), _ptr(frm), _ptr(to), _ptr(place), _stream()),
            "dash_compact_pages")
    return (new_refs, new_table, frm, to) if n > 1 else (new_refs, new_table, frm[:0], to[:0])


class PagePool:
    """The pages of a serving batch: ``caches`` (PageCaches), and for `rows` sequences of at most
    `max_pages` pages the state refs, table and lens.  Every method enqueues its launches and
    returns; those that can fail return ``ok`` (int32 [1] on the GPU), 0 where nothing changed.
    The state tensors stay the same objects, so a captured graph may read them, until compact()
    writes the new state into them."""

    def __init__(self, caches, rows, max_pages):
        if rows > MAX_ROWS:
            raise NotImplementedError(f"tables of at most {MAX_ROWS} rows")
        self.caches = caches
        self.page_size = caches.page_size
        dev = caches.device
        self.refs = torch.zeros(caches.num_pages, dtype=torch.int32, device=dev)
        self.table = torch.full((rows, max_pages), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)

    def reserve(self, new_lens):
        """Room for new_lens [rows] tokens (reserve_pages), shared last pages copied."""
        ok, frm, to = reserve_pages(self.refs, self.table, self.lens, new_lens, self.page_size)
        copy_pages(self.caches, frm, to)
        return ok

    def fork(self, src, dst):
        """The empty rows dst become the rows src (fork_pages), their last pages copied.  Rows are
        forked between steps: what reserve() gave a row for a step counts as its tokens until keep()."""
        ok, frm, to = fork_pages(self.refs, self.table, self.lens, src, dst, self.page_size)
        copy_pages(self.caches, frm, to)
        return ok

    def free(self, keep_lens):
        """Rows cut to keep_lens [rows] tokens (free_pages)."""
        free_pages(self.refs, self.table, self.lens, keep_lens, self.page_size)

    def keep(self, path, count, context_lens):
        """After a verification of the rows' trees (path and count of tree.verify_tree; a row
        without nodes has count 0 and stays): the accepted rows moved up, the rest given back.
        A row that does not hold the slots of its accepted nodes, as after a reserve that was
        refused, stays as it is: none of them stands.  Returns the rows' tokens [rows] int32."""
        return self._keep(path, count, context_lens)[1]

    def _keep(self, path, count, context_lens):
        step = _keep_lens(path, count, context_lens, self.lens)
        keep_rows(self.caches, path, step[0], context_lens, self.table)
        self.free(step[1])
        return step

    def reserve_step(self, query_lens, rows):
        """Room for query_lens [rows of the pool] new tokens (a number below 0 counts as 0) of a step whose
        batch has `rows` rows.  Returns (ok, context_lens, query_lens): the tokens of every row before,
        and the new ones.  ok is 0, and nothing changed, where the pool has no room or the batch has
        fewer rows than there are new tokens."""
        rows = int(rows)
        if not 0 <= rows < 2 ** 31:
            raise ValueError(f"a batch of {rows} rows")
        _shape(query_lens, self.lens.shape, "query_lens")
        if self.table.shape[1] * self.page_size > MAX_STEP_TOKENS:
            raise NotImplementedError("steps over tables of at most 2^31 - 2 tokens a row")
        with _device(self.lens, query_lens):
            R, n = self.lens.numel(), _i32(query_lens)
            new, ctx, want = _ints(n.device, R, R, R)
            _lib.check(_lib.load().dash_step_lens(_ptr(n), _ptr(self.lens), R, rows, _ptr(new), _ptr(ctx),
                                                  _ptr(want), _stream()), "dash_step_lens")
            return self.reserve(want), ctx, new

    def step_rows(self, context_lens, query_lens, rows):
        """(cu_seqlens_q, seq, positions, slots) of a step's new tokens (step_rows), once reserve()
        has made room for them: rows that hold no slot for a token get -1 for it."""
        return step_rows(self.table, context_lens, query_lens, self.page_size,
                         self.caches.num_pages, rows, self.lens)

    def compact(self):
        """The pages in use moved to the lowest numbers, in the caches too."""
        refs, table, frm, to = compact_pages(self.refs, self.table, self.lens, self.page_size)
        copy_pages(self.caches, frm, to)
        self.refs.copy_(refs)
        self.table.copy_(table)
