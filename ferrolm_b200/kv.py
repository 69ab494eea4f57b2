"""The key/value cache of a language model as an index over its blocks.

`KvCache` stands beside `FlatIndex`, `IvfPq` and `Hnsw`: rows are added, read back and searched by inner product.  The rows
are a model's keys and values; they lie in pages, one page to a block of a sequence, in 16 bits or rounded to 8; a search
finds for every query the blocks that promise the largest inner products; and what is wanted of the blocks found, or of
all of them, is attention.

A call is about a batch: `table[b, i]` is the page of block i of sequence b, `lens[b]` the sequence's rows, those of the call
among them, and the call is about its last ones.  Row i of the n that sequence b brings stands at position
`lens[b] - n + i` and is row `cu[b] + i` of the call's tensors; without `cu` every sequence brings one row.  Rows before
`cu[0]` and from `cu[-1]` on belong to no sequence (a padded batch): they are not read, and what a result holds there is what was there
before.  Positions below 0 or in a block that the table has no column for, and blocks whose table entry is not a page of the
cache (-1, say), are skipped: nothing is written or read there and nothing attends to them.

The calls run on the current torch stream of the cache's device and do not wait for it; they can be captured into a CUDA
graph.  Tensors are used on that stream only.  They know no gradients, in neither mode.  A length below 0 counts as 0.
"""
from __future__ import annotations

import ctypes as C

from ._lib import FV_ERR_ARG, FerrovecError, check, fv_kv, fv_kv_batch, lib

KINDS = {"same": 0, "int8": 1, "e4m3": 2, "int4x32": 4}


def _refuse(text: str):
    raise FerrovecError(FV_ERR_ARG, text)


class KvCache:
    """Pages of keys and values for `heads` key heads of `dim` (64, 96 or 128) components.

    `kind`: "same" keeps rows as they come (`dtype`: torch.bfloat16 or torch.float16); "int8" and "e4m3" round every row
    of a head to 8 bits with a scale of its own (max |x| / 127 or / 448).  A row with a value that is not finite reads
    back as NaN from an 8-bit cache.  "int4x32" rounds to 4 bits, whole numbers from -7 to 7, with a scale for every 32
    neighbouring components: max |x| / 7 rounded up to a number of 4 significant bits, from 2**-17 to 9216, so that what a row
    holds is exact in `dtype`; components beyond 64512 become that, and a group with a value that is not finite reads back
    as NaN.  `page_size`: 16, 32, 64 or 128 rows.

    The memory is torch's: `k`, `v` (pages, heads, page_size, dim), `k_scale`, `v_scale` (pages, heads, page_size) or None (of
    "int4x32" bytes: (..., dim / 2), two codes each, and (..., dim / 32); `include/ferrovec.h` says which component is where),
    `bounds` (pages, heads, 2, dim: the componentwise minima and maxima of a block's keys), `bound_codes` (the same in 8
    bits) and `bound_scale` (pages, heads).  `buffers`: a dict of them by these names, where the caller has them already.
    Their contents are anyone's to change; the tensors are the cache's for good, since every call goes to their addresses.
    """

    def __init__(self, pages: int, heads: int, dim: int, page_size: int = 64, dtype=None, kind: str = "same", device=None,
                 buffers: dict | None = None):
        import torch

        dtype = torch.bfloat16 if dtype is None else dtype
        if kind not in KINDS:
            _refuse(f"kind is one of {', '.join(KINDS)}: got {kind!r}")
        if dtype not in (torch.bfloat16, torch.float16):
            _refuse(f"dtype is torch.bfloat16 or torch.float16: got {dtype}")
        if pages < 0 or heads < 1 or dim not in (64, 96, 128) or page_size not in (16, 32, 64, 128):
            _refuse(f"pages >= 0, heads >= 1, dim 64, 96 or 128, page_size 16, 32, 64 or 128: got {pages}, {heads}, {dim}, {page_size}")
        self.pages, self.heads, self.dim, self.page_size, self.dtype, self.kind = pages, heads, dim, page_size, dtype, kind
        held = {"same": dtype, "int8": torch.int8, "e4m3": torch.float8_e4m3fn, "int4x32": torch.uint8}[kind]
        rows, scales, scale = (pages, heads, page_size, dim), (pages, heads, page_size), torch.float32
        if kind == "int4x32":
            rows, scales, scale = (pages, heads, page_size, dim // 2), (pages, heads, page_size, dim // 32), torch.uint8
        want = {"k": (rows, held), "v": (rows, held), "bounds": ((pages, heads, 2, dim), dtype),
                "bound_codes": ((pages, heads, 2, dim), torch.int8), "bound_scale": ((pages, heads), torch.float32)}
        if kind != "same":
            want |= {"k_scale": (scales, scale), "v_scale": (scales, scale)}
        if buffers is None:
            device = torch.device("cuda" if device is None else device)
            buffers = {n: torch.zeros(s, dtype=t, device=device) for n, (s, t) in want.items()}
        for name, (shape, t) in want.items():
            x = buffers.get(name)
            if x is None or tuple(x.shape) != shape or x.dtype != t or not x.is_contiguous():
                _refuse(f"buffers[{name!r}] is a contiguous {t} tensor of {shape}")
        self._held = {n: buffers[n] for n in want}
        if not self.k.is_cuda or any(buffers[n].device != self.k.device for n in want):
            _refuse("the buffers of a cache are on one CUDA device")
        self.device = self.k.device
        at = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
        self._c = fv_kv(self.device.index, int(dtype == torch.float16), KINDS[kind], page_size, heads, dim, pages, at(self.k),
                        at(self.v), at(self.k_scale), at(self.v_scale), at(self.bounds), at(self.bound_codes), at(self.bound_scale))
        self._ready()

    def _ready(self):
        """What every call uses, looked up once."""
        import torch

        L = lib()
        self._ref, self._i32, self._f32, self._index = C.byref(self._c), torch.int32, torch.float32, self.device.index
        self._grad, self._dual = torch.is_grad_enabled, torch.autograd.forward_ad
        self._empty_like, self._contiguous = torch.empty_like, torch.contiguous_format
        self._get_stream, self._work_sizes = torch._C._cuda_getCurrentRawStream, {}
        self._add, self._vectors, self._search, self._attend = L.fv_kv_add_dev, L.fv_kv_vectors_dev, L.fv_kv_search_dev, L.fv_kv_attend_dev
        self._copy = L.fv_kv_copy_pages_dev

    k, v, bounds, bound_codes, bound_scale, k_scale, v_scale = (
        property(lambda self, name=name: self._held.get(name)) for name in ("k", "v", "bounds", "bound_codes", "bound_scale", "k_scale", "v_scale"))

    # ---- the batch and the rows of a call
    def _batch(self, table, lens, cu, rows: int):
        i32, dev = self._i32, self.device
        if table.dtype is not i32 or lens.dtype is not i32 or table.device != dev or lens.device != dev or table.dim() != 2:
            _refuse("table (sequences, blocks) and lens are int32 tensors on the cache's device")
        n, width = table.shape
        stride, next_one = table.stride()
        if lens.dim() != 1 or len(lens) != n or not lens.is_contiguous() or next_one != 1 and width > 1:
            _refuse("lens is contiguous and has an entry for each row of table, and rows of table are contiguous")
        at = None
        if cu is not None:
            if cu.dtype is not i32 or cu.device != dev or cu.dim() != 1 or len(cu) != n + 1 or not cu.is_contiguous():
                _refuse("cu is a contiguous int32 tensor on the cache's device, with one entry more than there are sequences")
            at = cu.data_ptr()
        elif rows != n:
            _refuse(f"without cu every sequence brings one row: got {rows} rows for {n} sequences")
        return fv_kv_batch(table.data_ptr(), stride, width, lens.data_ptr(), at, n, rows)

    def _rows(self, x, what: str, heads: int):
        """(rows, heads, dim) with any strides of whole 16 bytes, copied where it is not like that: it, its address, strides and
        rows.  `heads`: 0 for any."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.dim or heads and shape[1] != heads:
            _refuse(f"{what} is (rows, heads, dim) with dim {self.dim}" + (f" and {heads} heads" if heads else "") + f": got {tuple(shape)}")
        if x.dtype is not self.dtype or x.device != self.device:
            _refuse(f"{what} is {self.dtype} on {self.device}: got {x.dtype} on {x.device}")
        if x.requires_grad and self._grad():
            _refuse(f"{what} wants a gradient, and the cache gives none: call it under torch.no_grad() or with a detached tensor")
        if self._dual._current_level >= 0 and self._dual.unpack_dual(x).tangent is not None:
            _refuse(f"{what} has a tangent, and the cache gives none: call it with the primal of unpack_dual")
        r, h, d = x.stride()
        at = x.data_ptr()
        if d != 1 or (r | h) & 7 or at & 15:
            x = x.clone(memory_format=self._contiguous)
            r, h, d = x.stride()
            at = x.data_ptr()
        return x, at, r, h, shape[0]

    # ---- rows
    def add(self, k, v, table, lens, cu=None):
        """Writes the call's rows `k` and `v` (rows, heads, dim) into their pages and keeps the bounds of their blocks.

        A page that is written to is one block of one sequence of the call.  A block that gets its first row forgets what its
        bounds were; one that is written again from its middle on keeps the bounds of the rows that were there.  Key
        components that are not finite count as zero in the bounds."""
        k, kp, kr, kh, rows = self._rows(k, "k", self.heads)
        v, vp, vr, vh, more = self._rows(v, "v", self.heads)
        if rows != more:
            _refuse(f"k and v have as many rows: got {rows} and {more}")
        status = self._add(self._ref, self._get_stream(self._index), self._batch(table, lens, cu, rows), kp, kr, kh, vp, vr, vh)
        if status:
            check(status)

    def vectors(self, table, lens, cu=None, rows: int | None = None, out=None):
        """The last rows of every sequence as the cache holds them: (k, v), each (rows, heads, dim) of `dtype`.

        `rows`: how many rows the call has; without it cu[-1] is read, for which the host waits.  `out`: the two tensors to
        write to; what stands for no row of the cache stays as it was in them."""
        if rows is None:
            rows = table.shape[0] if cu is None else int(cu[-1]) if out is None else out[0].shape[0]
        shape = (rows, self.heads, self.dim)
        if out is None:
            k, v = self.bounds.new_empty(shape), self.bounds.new_empty(shape)
        else:
            k, v = out
            self._check_out(k, shape)
            self._check_out(v, shape)
        status = self._vectors(self._ref, self._get_stream(self._index), self._batch(table, lens, cu, rows), k.data_ptr(), v.data_ptr())
        if status:
            check(status)
        return k, v

    def copy_pages(self, src, dst):
        """Copies page `src[i]` to `dst[i]`, rows, scales and bounds (int32 tensors of one length).  No page is twice in `dst`, or in both; pairs
        with a number that is no page are skipped.  `KvPages` does this where sequences share pages."""
        for x in (src, dst):
            if x.dtype is not self._i32 or x.device != self.device or x.dim() != 1 or not x.is_contiguous() or len(x) != len(src):
                _refuse(f"src and dst are contiguous int32 tensors of one length on {self.device}")
        status = self._copy(self._ref, self._get_stream(self._index), src.data_ptr(), dst.data_ptr(), len(src), None)
        if status:
            check(status)

    def _check_out(self, x, shape):
        if tuple(x.shape) != shape or x.dtype is not self.dtype or x.device != self.device or not x.is_contiguous() or x.data_ptr() & 15:
            _refuse(f"what is written to is a contiguous {self.dtype} tensor of {shape} on {self.device}")

    # ---- search
    def search_blocks(self, q, table, lens, k: int, cu=None, first: int = 1, recent: int = 2, out=None):
        """For every row of the call and key head the `k` blocks that promise the queries the largest inner products:
        (rows, heads, k) int32, ascending, -1 behind the last.

        `q` is (rows, heads * group, dim), the query heads of a key head one behind the other.  A block's score is the sum
        over those heads of the largest inner product that the block's bounds allow, worked out in whole numbers, so that
        it does not depend on how the work is cut; of equal scores the lower block is taken.  Queries (with one scale for a
        key head's group) and bounds are rounded to 8 bits for that, to nearest: a score is close to the bound, not always
        above it, and a head below 1/254 of its group's largest component counts as nothing.

        The first `first` blocks and the last `recent` ones up to the query's own are among the `k` before any other; of more
        than `k` such blocks the lowest are the result, and the query's own is not in it: `k` is to be at least
        `first + recent`.  Blocks behind the query's position and blocks without a page are never among them."""
        q, qp, qr, qh, rows = self._rows(q, "q", 0)
        group = self._group(q)
        if first < 0 or recent < 0 or k < 1:
            _refuse(f"k is 1 or more, first and recent are 0 or more: got {k}, {first}, {recent}")
        shape, batch = (rows, self.heads, k), self._batch(table, lens, cu, rows)
        if out is None:
            out = table.new_empty(shape)
        elif tuple(out.shape) != shape or out.dtype is not self._i32 or out.device != self.device or not out.is_contiguous():
            _refuse(f"out is a contiguous int32 tensor of {shape} on {self.device}")
        status = self._search(self._ref, self._get_stream(self._index), batch, qp, qr, qh, group, k, first, recent, out.data_ptr())
        if status:
            check(status)
        return out

    # ---- attention
    def attend(self, q, table, lens, cu=None, blocks=None, scale: float | None = None, return_lse: bool = False, out=None):
        """softmax(scale q k^T) v over the rows at and before each query's own position: (rows, heads * group, dim), and with
        `return_lse` also the natural logarithms of the sums, (rows, heads * group) float32.

        `blocks`: the blocks that each row and key head attends to, (rows, heads, k) int32 as `search_blocks` gives them;
        without it, all of them.  Entries that are no block the query can see, and entries not above all of those before
        them, are skipped.  A row with nothing to attend to gets zeros and -inf.  `scale` is dim ** -0.5 unless given.
        `out`: the tensor to write to (with `return_lse` a pair).

        Calls whose sequences bring more than four rows on average are worked on as prompts, others row by row (as is a
        prompt whose table has more than about 16,400 columns); a long prompt is faster in a call of its own than among
        many single rows."""
        q, qp, qr, qh, rows = self._rows(q, "q", 0)
        heads, group, at, k = q.shape[1], self._group(q), None, 0
        if blocks is not None:
            shape = blocks.shape
            if blocks.dtype is not self._i32 or blocks.device != self.device or len(shape) != 3 or shape[0] != rows or shape[1] != self.heads or not blocks.is_contiguous():
                _refuse(f"blocks is a contiguous int32 tensor of ({rows}, {self.heads}, k) on {self.device}")
            at, k = blocks.data_ptr(), shape[2]
            if k == 0:
                _refuse("blocks has no entry for a row; leave it out to attend to all blocks")
        lse = lse_at = None
        if out is None:
            out = self._empty_like(q, memory_format=self._contiguous)
            if return_lse:
                lse = self.bound_scale.new_empty((rows, heads))
        else:
            out, lse = out if return_lse else (out, None)
            self._check_out(out, (rows, heads, self.dim))
            if return_lse and (tuple(lse.shape) != (rows, heads) or lse.dtype is not self._f32 or lse.device != self.device or not lse.is_contiguous()):
                _refuse(f"lse is a contiguous float32 tensor of {(rows, heads)} on {self.device}")
        if return_lse:
            lse_at = lse.data_ptr()
        batch, work_at = self._batch(table, lens, cu, rows), None
        shape = rows, heads, batch.nseq, batch.table_width
        size = self._work_sizes.get(shape)  # depends on these alone
        if size is None:
            if len(self._work_sizes) > 4096:
                self._work_sizes.clear()
            size = self._work_sizes[shape] = lib().fv_kv_attend_work(self._ref, batch, group)
        if size:
            work = self.bound_scale.new_empty(size >> 2)
            work_at = work.data_ptr()
        status = self._attend(self._ref, self._get_stream(self._index), batch, qp, qr, qh, group, at, k, self.dim**-0.5 if scale is None else scale,
                              out.data_ptr(), lse_at, work_at, size)
        if status:
            check(status)
        return (out, lse) if return_lse else out

    def _group(self, q) -> int:
        group, more = divmod(q.shape[1], self.heads)
        if more or not group:
            _refuse(f"q has a multiple of the cache's {self.heads} heads: got {q.shape[1]}")
        return group


__all__ = ["KvCache"]
