"""The key/value cache of a language model as an index over its blocks.

`KvCache` stands beside `FlatIndex`, `IvfPq` and `Hnsw`: rows are added, read back and searched by inner product.  The rows
are a model's keys and values; they lie in pages, one page to a block of a sequence, in 16 bits or rounded to 8; a search
finds for every query the blocks that promise the largest inner products; and what is wanted of the blocks found, or of
all of them, is attention.

A call is about a batch: `table[b, i]` is the page of block i of sequence b, `lens[b]` the sequence's rows, those of the call
among them, and the call is about its last ones.  Row i of the n that sequence b brings stands at position
`lens[b] - n + i` and is row `cu[b] + i` of the call's tensors; without `cu` every sequence brings one row.  Rows from
`cu[-1]` on belong to no sequence (a padded batch): they are not read, and what a result holds there is what was there
before.  Positions below 0 or in a block that the table has no column for, and blocks whose table entry is not a page of the
cache (-1, say), are skipped: nothing is written or read there and nothing attends to them.

The calls run on the current torch stream of the cache's device and do not wait for it; they can be captured into a CUDA
graph.  Tensors are used on that stream only.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import FV_ERR_ARG, FerrovecError, check, fv_kv, fv_kv_batch, lib

KINDS = ("same", "int8", "e4m3")


def _refuse(text: str):
    raise FerrovecError(FV_ERR_ARG, text)


class KvCache:
    """Pages of keys and values for `heads` key heads of `dim` (64, 96 or 128) components.

    `kind`: "same" keeps rows as they come (`dtype`: torch.bfloat16 or torch.float16); "int8" and "e4m3" round every row
    of a head to 8 bits with a scale of its own (max |x| / 127 or / 448).  A row with a value that is not finite reads
    back as NaN from an 8-bit cache.  `page_size`: 16, 32, 64 or 128 rows.

    The memory is torch's: `k`, `v` (pages, heads, page_size, dim), `k_scale`, `v_scale` (pages, heads, page_size) or None,
    `bounds` (pages, heads, 2, dim: the componentwise minima and maxima of a block's keys), `bound_codes` (the same in 8
    bits) and `bound_scale` (pages, heads).  `buffers`: a dict of them by these names, where the caller has them already.
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
        held = {"same": dtype, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}[kind]
        rows, scales = (pages, heads, page_size, dim), (pages, heads, page_size)
        want = {"k": (rows, held), "v": (rows, held), "bounds": ((pages, heads, 2, dim), dtype),
                "bound_codes": ((pages, heads, 2, dim), torch.int8), "bound_scale": ((pages, heads), torch.float32)}
        if kind != "same":
            want |= {"k_scale": (scales, torch.float32), "v_scale": (scales, torch.float32)}
        if buffers is None:
            device = torch.device("cuda" if device is None else device)
            buffers = {n: torch.zeros(s, dtype=t, device=device) for n, (s, t) in want.items()}
        for name, (shape, t) in want.items():
            x = buffers.get(name)
            if x is None or tuple(x.shape) != shape or x.dtype != t or not x.is_contiguous():
                _refuse(f"buffers[{name!r}] is a contiguous {t} tensor of {shape}")
        self.k, self.v, self.bounds = buffers["k"], buffers["v"], buffers["bounds"]
        self.bound_codes, self.bound_scale = buffers["bound_codes"], buffers["bound_scale"]
        self.k_scale, self.v_scale = (buffers["k_scale"], buffers["v_scale"]) if kind != "same" else (None, None)
        if not self.k.is_cuda or any(buffers[n].device != self.k.device for n in want):
            _refuse("the buffers of a cache are on one CUDA device")
        self.device = self.k.device
        at = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
        self._c = fv_kv(self.device.index, int(dtype == torch.float16), KINDS.index(kind), page_size, heads, dim, pages, at(self.k),
                        at(self.v), at(self.k_scale), at(self.v_scale), at(self.bounds), at(self.bound_codes), at(self.bound_scale))
        self._ref = C.byref(self._c)
        self._i32, self._get_stream = torch.int32, torch._C._cuda_getCurrentRawStream

    # ---- the batch and the rows of a call
    def _batch(self, table, lens, cu, rows: int):
        i32, dev = self._i32, self.device
        if table.dtype != i32 or lens.dtype != i32 or table.device != dev or lens.device != dev or table.dim() != 2:
            _refuse("table (sequences, blocks) and lens are int32 tensors on the cache's device")
        n, width = table.shape
        if lens.shape != (n,) or lens.stride(0) != 1 and n > 1 or table.stride(1) != 1 and width > 1 or table.stride(0) < 0:
            _refuse("lens has an entry for each row of table, and rows of table are contiguous")
        at = None
        if cu is not None:
            if cu.dtype != i32 or cu.device != dev or cu.shape != (n + 1,) or not cu.is_contiguous():
                _refuse("cu is a contiguous int32 tensor on the cache's device, with one entry more than there are sequences")
            at = cu.data_ptr()
        elif rows != n:
            _refuse(f"without cu every sequence brings one row: got {rows} rows for {n} sequences")
        return C.byref(fv_kv_batch(table.data_ptr(), table.stride(0), width, lens.data_ptr(), at, n, rows))

    def _rows(self, x, what: str, heads: int | None = None):
        """(rows, heads, dim) with any strides of whole 16 bytes; copied where it is not like that."""
        if x.dim() != 3 or x.shape[2] != self.dim or heads is not None and x.shape[1] != heads:
            _refuse(f"{what} is (rows, heads, dim) with dim {self.dim}" + (f" and {heads} heads" if heads is not None else "") + f": got {tuple(x.shape)}")
        if x.dtype != self.dtype or x.device != self.device:
            _refuse(f"{what} is {self.dtype} on {self.device}: got {x.dtype} on {x.device}")
        r, h, d = x.stride()
        if d != 1 or (r | h) & 7 or r < 0 or h < 0 or x.data_ptr() & 15:
            x = x.clone(memory_format=_contiguous())
            r, h, d = x.stride()
        return x, x.data_ptr(), r, h

    def _stream(self) -> int:
        return self._get_stream(self.device.index)

    # ---- rows
    def add(self, k, v, table, lens, cu=None):
        """Writes the call's rows `k` and `v` (rows, heads, dim) into their pages and keeps the bounds of their blocks.

        A page that is written to belongs to one sequence of the call.  A block that gets its first row forgets what its
        bounds were; one that is written again from its middle on keeps the bounds of the rows that were there.  Key
        components that are not finite count as zero in the bounds."""
        k, kp, kr, kh = self._rows(k, "k", self.heads)
        v, vp, vr, vh = self._rows(v, "v", self.heads)
        if k.shape != v.shape:
            _refuse(f"k and v have as many rows: got {k.shape[0]} and {v.shape[0]}")
        check(lib().fv_kv_add_dev(self._ref, self._stream(), self._batch(table, lens, cu, k.shape[0]), kp, kr, kh, vp, vr, vh))

    def vectors(self, table, lens, cu=None, rows: int | None = None, out=None):
        """The last rows of every sequence as the cache holds them: (k, v), each (rows, heads, dim) of `dtype`.

        `rows`: how many rows the call has; without it cu[-1] is read, for which the host waits.  `out`: the two tensors to
        write to; what stands for no row of the cache stays as it was in them."""
        import torch

        if rows is None:
            rows = table.shape[0] if cu is None else int(cu[-1]) if out is None else out[0].shape[0]
        if out is None:
            k, v = torch.empty((2, rows, self.heads, self.dim), dtype=self.dtype, device=self.device).unbind(0)
        else:
            k, v = out
            for x in out:
                if tuple(x.shape) != (rows, self.heads, self.dim) or x.dtype != self.dtype or x.device != self.device or not x.is_contiguous() or x.data_ptr() & 15:
                    _refuse(f"out is two contiguous {self.dtype} tensors of {(rows, self.heads, self.dim)} on {self.device}")
        check(lib().fv_kv_vectors_dev(self._ref, self._stream(), self._batch(table, lens, cu, rows), k.data_ptr(), v.data_ptr()))
        return k, v

    # ---- search
    def search_blocks(self, q, table, lens, k: int, cu=None, first: int = 1, recent: int = 2, out=None):
        """For every row of the call and key head the `k` blocks that promise the queries the largest inner products:
        (rows, heads, k) int32, ascending, -1 behind the last.

        `q` is (rows, heads * group, dim), the query heads of a key head one behind the other.  A block's score is the sum
        over those heads of the largest inner product that the block's bounds allow, worked out in whole numbers, so that
        it does not depend on how the work is cut; of equal scores the lower block is taken.  The first `first` blocks
        and the last `recent` ones up to the query's own are always among the `k`, blocks behind the query's position and
        blocks without a page never."""
        import torch

        q, qp, qr, qh = self._rows(q, "q")
        rows, group = q.shape[0], self._group(q)
        if first < 0 or recent < 0 or k < 1:
            _refuse(f"k is 1 or more, first and recent are 0 or more: got {k}, {first}, {recent}")
        shape = (rows, self.heads, k)
        if out is None:
            out = torch.empty(shape, dtype=self._i32, device=self.device)
        elif tuple(out.shape) != shape or out.dtype != self._i32 or out.device != self.device or not out.is_contiguous():
            _refuse(f"out is a contiguous int32 tensor of {shape} on {self.device}")
        check(lib().fv_kv_search_dev(self._ref, self._stream(), self._batch(table, lens, cu, rows), qp, qr, qh, group, k, first, recent, out.data_ptr()))
        return out

    # ---- attention
    def attend(self, q, table, lens, cu=None, blocks=None, scale: float | None = None, return_lse: bool = False, out=None):
        """softmax(scale q k^T) v over the rows at and before each query's own position: (rows, heads * group, dim), and with
        `return_lse` also the natural logarithms of the sums, (rows, heads * group) float32.

        `blocks`: the blocks that each row and key head attends to, (rows, heads, k) int32 as `search_blocks` gives them;
        without it, all of them.  Entries that are no block the query can see, and entries not above all of those before
        them, are skipped.  A row with nothing to attend to gets zeros and -inf.  `scale` is dim ** -0.5 unless given.
        `out`: the tensor to write to (with `return_lse` a pair)."""
        import torch

        q, qp, qr, qh = self._rows(q, "q")
        rows, heads = q.shape[0], q.shape[1]
        group, at, k = self._group(q), None, 0
        if blocks is not None:
            if blocks.dtype != self._i32 or blocks.device != self.device or blocks.dim() != 3 or tuple(blocks.shape[:2]) != (rows, self.heads) or not blocks.is_contiguous():
                _refuse(f"blocks is a contiguous int32 tensor of ({rows}, {self.heads}, k) on {self.device}")
            at, k = blocks.data_ptr(), blocks.shape[2]
            if k == 0:
                _refuse("blocks has no entry for a row; leave it out to attend to all blocks")
        lse = None
        if out is None:
            out = torch.empty((rows, heads, self.dim), dtype=self.dtype, device=self.device)
            if return_lse:
                lse = torch.empty((rows, heads), dtype=torch.float32, device=self.device)
        else:
            out, lse = out if return_lse else (out, None)
            if tuple(out.shape) != (rows, heads, self.dim) or out.dtype != self.dtype or out.device != self.device or not out.is_contiguous() or out.data_ptr() & 15:
                _refuse(f"out is a contiguous {self.dtype} tensor of {(rows, heads, self.dim)} on {self.device}")
            if return_lse and (tuple(lse.shape) != (rows, heads) or lse.dtype != torch.float32 or lse.device != self.device or not lse.is_contiguous()):
                _refuse(f"lse is a contiguous float32 tensor of {(rows, heads)} on {self.device}")
        batch = self._batch(table, lens, cu, rows)
        size, work = lib().fv_kv_attend_work(self._ref, batch, group), None
        if size:
            work = torch.empty(size, dtype=torch.uint8, device=self.device)
        check(lib().fv_kv_attend_dev(self._ref, self._stream(), batch, qp, qr, qh, group, at, k, self.dim**-0.5 if scale is None else scale,
                                     out.data_ptr(), None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), size))
        return (out, lse) if return_lse else out

    def _group(self, q) -> int:
        group, more = divmod(q.shape[1], self.heads)
        if more or not group:
            _refuse(f"q has a multiple of the cache's {self.heads} heads: got {q.shape[1]}")
        return group


def _contiguous():
    import torch

    return torch.contiguous_format


__all__ = ["KvCache"]
