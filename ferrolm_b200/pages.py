"""Which pages of a key/value cache are in use, and by how many sequences.

A `KvCache` takes its pages from a table that the caller keeps.  `KvPages` counts for every page how many entries of tables
hold it, so that sequences can share the pages of their common rows: samples or beams of one request, requests with the same beginning.

    pages = fv.KvPages(caches)                       # the caches of a model's layers: their rows lie in the same pages
    pages.extend(table, lens, more)                  # room for the next rows; a page that others hold as well is copied first
    children = pages.fork(table, lens, parents)      # sequences that go on from others
    pages.free(table)                                # pages given back; with lens, those behind that many rows (drafts not taken)
    pages.compact(table, children)                   # pages in use moved to the front of the memory

Everything happens on the GPU, on the current torch stream, without waiting, and can be captured into a graph.  Calls on one
`KvPages` change its counts and follow one another on one stream (or wait for one another).  `table` is (sequences, blocks) int32,
an entry outside of 0 .. pages - 1 (-1, say) is none; `lens`, `more` and `parents` are int32.  A length below 0 counts as 0.
"""
from __future__ import annotations

import ctypes as C

from ._lib import check, fv_pages, fv_table, lib
from .kv import KvCache, _refuse


def _shared(a: fv_table, b: fv_table) -> int:
    """How many of a's entries are entries of b too.  Rows of a table do not overlap one another."""
    size = lambda t: 4 * ((t.nseq - 1) * t.stride + t.width) if t.nseq and t.width else 0  # noqa: E731
    begin_a, begin_b = a.table or 0, b.table or 0
    if not size(a) or not size(b) or begin_a + size(a) <= begin_b or begin_b + size(b) <= begin_a:
        return 0
    if (begin_a, a.stride, a.width, a.nseq) == (begin_b, b.stride, b.width, b.nseq):
        return a.nseq * a.width
    begin, found = (begin_a - begin_b) // 4, 0  # of a, in b
    if a.stride == b.stride and a.nseq > 1 and b.nseq > 1:  # row i of a begins in row i + k of b, and may end in the next one
        k, at = divmod(begin, b.stride)
        rows = lambda k: max(min(a.nseq, b.nseq - k) - max(-k, 0), 0)  # noqa: E731
        return rows(k) * max(min(a.width, b.width - at), 0) + rows(k + 1) * max(min(at + a.width - b.stride, b.width), 0)
    for i in range(a.nseq):
        row = begin + i * a.stride
        step = b.stride if b.nseq > 1 else max(b.stride, row + a.width + b.width, 1)
        j = max((row - b.width) // step, 0)
        while j < b.nseq and j * step < row + a.width:
            found += max(min(row + a.width, j * step + b.width) - max(row, j * step), 0)
            j += 1
    return found


class KvPages:
    """The pages of one cache or of several that share a table (a model's layers).

    `refs` (pages,) int32: how many entries of tables hold a page; 0: it is free.  The caller may write to it, to set aside
    pages of its own or to begin from tables that exist.  `refs=`: the tensor to use.
    `missing`, a number on the GPU (int32): how many pages the last `extend` lacked; where it is not 0, that call changed nothing.
    `used`, another: the pages in use when `compact` was called last."""

    def __init__(self, caches, refs=None):
        import torch

        self.caches = (caches,) if isinstance(caches, KvCache) else tuple(caches)
        if not self.caches or not all(isinstance(c, KvCache) for c in self.caches):
            _refuse("caches is a KvCache or several of them")
        first = self.caches[0]
        self.pages, self.page_size, self.device = first.pages, first.page_size, first.device
        if any((c.pages, c.page_size, c.device) != (self.pages, self.page_size, self.device) for c in self.caches):
            _refuse("the caches have as many pages as one another, of the same size, on one device")
        if refs is None:
            refs = torch.zeros(self.pages, dtype=torch.int32, device=self.device)
        if refs.dtype is not torch.int32 or refs.device != self.device or tuple(refs.shape) != (self.pages,) or not refs.is_contiguous():
            _refuse(f"refs is a contiguous int32 tensor of ({self.pages},) on {self.device}")
        self._refs, self._i32 = refs, torch.int32
        self.missing, self.used = torch.zeros(2, dtype=torch.int32, device=self.device).unbind()
        self._c = fv_pages(self.device.index, self.page_size, self.pages, refs.data_ptr())
        self._ref, self._index, self._get_stream = C.byref(self._c), self.device.index, torch._C._cuda_getCurrentRawStream
        self._handles = (C.c_void_p * len(self.caches))(*(C.addressof(c._c) for c in self.caches))
        self._lib = lib()
        self._none = C.byref(fv_pages(self.device.index, self.page_size, 0, None))  # a call on no pages checks its table and does nothing
        self._compact_work, self._extend_work = self._lib.fv_pages_compact_work(self._ref), {}

    refs = property(lambda self: self._refs)

    def _table(self, table, what: str = "table"):
        if table.dtype is not self._i32 or table.device != self.device or table.dim() != 2:
            _refuse(f"{what} is an int32 tensor (sequences, blocks) on the caches' device")
        n, width = table.shape
        stride, next_one = table.stride()
        if (next_one != 1 and width > 1) or (stride < width and n > 1):
            _refuse(f"rows of {what} are contiguous, and do not overlap")
        return fv_table(table.data_ptr(), stride, width, n)

    def _numbers(self, x, n: int, what: str):
        if x.dtype is not self._i32 or x.device != self.device or tuple(x.shape) != (n,) or not x.is_contiguous():
            _refuse(f"{what} is a contiguous int32 tensor of ({n},) on the caches' device")
        return x.data_ptr()

    def fork(self, table, lens, parents, out=None):
        """A table whose row i is row `parents[i]` of `table`, up to the block of that row's last row (`lens`: those of `table`; None:
        the whole row), -1 behind it and everywhere where `parents[i]` is no row.  Pages are shared, not copied: every one counts
        once more.  `out`: the table to write to, which shares no entries with `table`; what it held is not given back."""
        t = self._table(table)
        at = None if lens is None else self._numbers(lens, t.nseq, "lens")
        if parents.dim() != 1:
            _refuse("parents is (sequences,)")
        by = self._numbers(parents, len(parents), "parents")
        if out is None:
            out = table.new_empty((len(parents), t.width))
        elif out.dim() != 2 or out.shape[0] != len(parents):
            _refuse(f"out has a row for each of the {len(parents)} parents")
        status = self._lib.fv_pages_fork_dev(self._ref, self._get_stream(self._index), t, at, by, self._table(out, "out"))
        if status:
            check(status)
        return out

    def free(self, table, lens=None):
        """Gives back the pages of the table's blocks (with `lens`, of those that begin at or behind that many rows): their entries become
        -1, and their pages count once less.  A page that nobody holds any more is free."""
        t = self._table(table)
        at = None if lens is None else self._numbers(lens, t.nseq, "lens")
        status = self._lib.fv_pages_free_dev(self._ref, self._get_stream(self._index), t, at)
        if status:
            check(status)

    def extend(self, table, lens, more):
        """Room for `more[b]` rows behind the `lens[b]` that sequence b has, in the table itself.

        Of the blocks from the one on that the first of those rows comes to, one without a page gets a free one, and one whose page others
        hold as well gets a free one with a copy of its rows, in every cache (a begun block also where `more[b]` is 0; below 0: the
        sequence is left as it is); where all who hold it are in this call, the first of them keeps it.  Free pages
        are taken in ascending order, for blocks in the table's order; a block that has a page of its own keeps it, so a call may be
        repeated.  Blocks behind the table's width get none.  If there are not enough free pages, nothing is changed and `missing`
        says how many were lacking."""
        t = self._table(table)
        at, by = self._numbers(lens, t.nseq, "lens"), self._numbers(more, t.nseq, "more")
        size = self._extend_work.get((t.nseq, t.width))
        if size is None:
            if len(self._extend_work) > 4096:
                self._extend_work.clear()
            size = self._extend_work[t.nseq, t.width] = self._lib.fv_pages_extend_work(self._ref, t)
        work = self._refs.new_empty(size >> 2)
        status = self._lib.fv_pages_extend_dev(self._ref, self._get_stream(self._index), self._handles, len(self.caches), t, at, by, self.missing.data_ptr(),
                                               work.data_ptr(), size)
        if status:
            check(status)

    @staticmethod
    def _once(tables):
        """Those of the tables that are no part of another: an entry is renumbered once."""
        inside = lambda a, b: _shared(a, b) == a.nseq * a.width  # noqa: E731
        keep = [a for i, a in enumerate(tables) if not any(inside(a, b) and not (i < j and inside(b, a)) for j, b in enumerate(tables) if j != i)]
        if any(_shared(a, b) for i, a in enumerate(keep) for b in keep[:i]):
            _refuse("tables share some of their entries: give what holds both, or parts that share none")
        return keep

    def compact(self, *tables):
        """Moves the n pages in use to 0 .. n - 1: those from n on go to the free ones below it, ascending to ascending, the others stay.
        The rows move in every cache, and the entries of `tables` become the pages' new numbers (-1 for a page that is free).  All
        tables that hold pages are to be among them; one that is part of another counts once, and others share no entries.  `used` becomes n."""
        each = [self._table(t) for t in tables]
        if len(each) > 1:
            each = self._once(each)
        stream = self._get_stream(self._index)
        for t in each:  # before anything moves
            status = self._lib.fv_pages_remap_dev(self._none, stream, None, t)
            if status:
                check(status)
        more = (self.pages + 3) // 4 * 4
        work = self._refs.new_empty((self._compact_work >> 2) + more)
        map_at = work.data_ptr() + self._compact_work
        status = self._lib.fv_pages_compact_dev(self._ref, stream, self._handles, len(self.caches), self.used.data_ptr(), map_at, work.data_ptr(), self._compact_work)
        for t in each:
            status = status or self._lib.fv_pages_remap_dev(self._ref, stream, map_at, t)
        if status:
            check(status)


__all__ = ["KvPages"]
