"""Rotary positions: queries and keys turned by where their rows stand, before they are added to a `KvCache` and attended to."""
from __future__ import annotations

import ctypes as C
import math
from decimal import Context, Decimal, localcontext

from ._lib import check, fv_rotary, fv_rotary_rows, lib
from .kv import _refuse

LAYOUTS = ("half", "pairs")


def _two_pi(digits: int) -> Decimal:
    """By Machin's formula, 4 (4 arctan(1/5) - arctan(1/239)) = pi."""
    with localcontext(Context(prec=digits + 10)):

        def arctan(inverse):
            power, total, k = Decimal(1) / inverse, Decimal(0), 1
            while power.adjusted() > -(digits + 8):
                total += power / k if k % 4 == 1 else -power / k
                power, k = power / (inverse * inverse), k + 2
            return total

        return 8 * (4 * arctan(5) - arctan(239))


DIGITS = 60
TWO_PI = _two_pi(DIGITS)


def _frequencies(base, part, factor, original, fast, slow) -> list[Decimal]:
    """w, to 55 digits and more."""
    with localcontext(Context(prec=DIGITS)):
        base, factor, fast, slow = (Decimal(float(x)) for x in (base, factor, fast, slow))
        step, w = (base.ln() * -2 / part).exp(), [Decimal(1)]
        while len(w) < part // 2:
            w.append(w[-1] * step)
        if original is None:
            return [x / factor for x in w]
        known = Decimal(float(original)) / TWO_PI
        kept = [min(max((known * x - slow) / (fast - slow), Decimal(0)), Decimal(1)) for x in w]
        return [x * (k + (1 - k) / factor) for x, k in zip(w, kept)]


def _turns(w: list[Decimal]) -> list[int]:
    """What pairs turn by at each position, in units of 2^-64 of a whole turn, to the nearest: a position of 31 bits is off by 2^-34 of a turn."""
    front = max(max(x.adjusted() for x in w), 0)  # digits in front of the point
    with localcontext(Context(prec=DIGITS + front)):
        unit = 2**64 / (_two_pi(DIGITS + front) if front else TWO_PI)
        return [int((x * unit).to_integral_value()) % 2**64 for x in w]


class Rotary:
    """Turns the first `part` of `dim` components in pairs, pair i by `position * w[i]` radians; the others stay as they are.

    `layout`: "half" pairs component i with i + part / 2, "pairs" 2 i with 2 i + 1.  dim and part (dim unless given) are multiples of 16.
    w[i] = base ** (-2 i / part).  For contexts that are `factor` times as long as those that a model was trained on: without
    `original` all w are divided by it; with `original`, the positions that the model was trained on, pairs that turn less than `slow`
    times in these are divided, those that turn more than `fast` times are not, those between are in part (the share that is kept grows
    linearly with the number of turns; where a checkpoint has it grow with the pair's index, give its `frequencies`), and what is turned is
    multiplied by `amplitude`, 0.1 ln(factor) + 1 unless given (1 without `original`, and for factors up to 1).  `frequencies` (part / 2
    numbers) are taken in place of all of that.  `dtype`: torch.bfloat16 or torch.float16, that of the rows.
    """

    def __init__(self, dim: int, part: int | None = None, layout: str = "half", base: float = 10000.0, factor: float = 1.0, original: int | None = None,
                 fast: float = 32.0, slow: float = 1.0, amplitude: float | None = None, frequencies=None, device=None):
        import torch

        part = dim if part is None else part
        if layout not in LAYOUTS:
            _refuse(f"layout is one of {', '.join(LAYOUTS)}: got {layout!r}")
        if dim < 16 or dim > 1024 or dim % 16 or part < 16 or part > dim or part % 16:
            _refuse(f"dim is a multiple of 16 up to 1024, part one up to dim: got {dim}, {part}")
        if not (base > 0 and factor > 0 and fast > slow and (original is None or original > 0)) or not all(map(math.isfinite, (base, factor, fast, slow))):
            _refuse(f"base, factor and original are above 0, and fast is above slow: got {base}, {factor}, {original}, {fast}, {slow}")
        if frequencies is not None:
            w = [float(x) for x in frequencies]
            if len(w) != part // 2 or not all(map(math.isfinite, w)):
                _refuse(f"frequencies are {part // 2} finite numbers")
            w = [Decimal(x) for x in w]
        else:
            w = _frequencies(base, part, factor, original, fast, slow)
            if not all(math.isfinite(float(x)) for x in w):
                _refuse(f"base {base} and factor {factor} make frequencies beyond what floats hold")
            if original is not None and amplitude is None and factor > 1:
                amplitude = 0.1 * math.log(factor) + 1.0
        amplitude = 1.0 if amplitude is None else float(amplitude)
        if not math.isfinite(amplitude):
            _refuse(f"amplitude is finite: got {amplitude}")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            _refuse("there is no CPU path")
        self.dim, self.part, self.layout, self.amplitude, self.frequencies = dim, part, layout, amplitude, tuple(map(float, w))
        self._turns = torch.tensor([x - 2**64 if x >= 2**63 else x for x in _turns(w)], dtype=torch.int64, device=device)
        self.device = self._turns.device
        at = self._turns.data_ptr()
        self._c = {t: C.pointer(fv_rotary(self.device.index, i, dim, part, LAYOUTS.index(layout), amplitude, at)) for i, t in enumerate((torch.bfloat16, torch.float16))}
        self._i32, self._contiguous, self._empty_like, self._index = torch.int32, torch.contiguous_format, torch.empty_like, self.device.index
        self._dual = torch.autograd.forward_ad
        self._grad, self._get_stream, self._rotate = torch.is_grad_enabled, torch._C._cuda_getCurrentRawStream, lib().fv_rotate_dev
        self._two = fv_rotary_rows * 2

    def _rows(self, x, out, dtype, rows: int, what: str):
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.dim or shape[0] != rows:
            _refuse(f"{what} is (rows, heads, {self.dim}), with as many rows as the others: got {tuple(shape)}")
        if x.dtype is not dtype or x.device != self.device:
            _refuse(f"{what} is {dtype} on {self.device}: got {x.dtype} on {x.device}")
        if x.requires_grad and self._grad():
            _refuse(f"{what} wants a gradient, and none is recorded: call it under torch.no_grad() or with a detached tensor, and turn gradients with back=True")
        if self._dual._current_level >= 0 and self._dual.unpack_dual(x).tangent is not None:
            _refuse(f"{what} has a tangent, and none is worked out: the turn is linear, so turn the tangent by itself")
        r, h, d = x.stride()
        at = x.data_ptr()
        if out is None:
            out = self._empty_like(x, memory_format=self._contiguous)
            to, tr, th = out.data_ptr(), shape[1] * self.dim, self.dim
        else:
            tr, th, td = out.stride() if out.dim() == 3 else (0, 0, 0)
            to = out.data_ptr()
            rows_span, head_span = (shape[0] - 1) * tr + self.dim, (shape[1] - 1) * th + self.dim  # of a head's rows, of a row's heads
            apart = (tr >= head_span or shape[0] < 2) and (th >= self.dim or shape[1] < 2) or (th >= rows_span or shape[1] < 2) and (tr >= self.dim or shape[0] < 2)
            if out.shape != shape or out.dtype is not dtype or out.device != self.device or td != 1 or (tr | th) & 7 or to & 15 or not apart:
                _refuse(f"what is written to is {dtype} of {tuple(shape)} on {self.device}, its rows on 16 bytes and apart from one another")
        if d != 1 or (r | h) & 7 or at & 15:
            x = x.clone(memory_format=self._contiguous)
            r, h, d = x.stride()
            at = x.data_ptr()
        return x, out, fv_rotary_rows(at, to, r, h, tr, th, shape[1])

    def rotate(self, q, k=None, lens=None, cu=None, positions=None, back: bool = False, out=None):
        """`q` (rows, heads, dim) turned, or with `k` (its heads may be others) both: (q, k).

        Rows stand where `KvCache`'s calls have them: the last of the `lens[b]` rows of sequence b, from row `cu[b]` on; without `cu` every
        sequence brings one row.  Or row i stands at `positions[i]`.  Rows of no sequence and positions below 0 are skipped: what the
        result holds there is what was there before.  `back` turns the other way: what undoes a turn (times amplitude ** 2), and what a
        gradient of the result becomes one of the rows by.  `out`: the tensors to write to, a pair with `k`; each may be the rows
        themselves, and otherwise overlaps neither those nor the other.  Sums are of 32 bits, and results are rounded once."""
        rows, dtype = q.shape[0] if q.dim() else 0, q.dtype
        c = self._c.get(dtype)
        if c is None:
            _refuse(f"rows are torch.bfloat16 or torch.float16: got {dtype}")
        lens_at = cu_at = pos_at = None
        n = 0
        if positions is not None:
            if lens is not None or cu is not None:
                _refuse("positions, or lens and cu")
            if positions.dtype is not self._i32 or positions.device != self.device or tuple(positions.shape) != (rows,) or not positions.is_contiguous():
                _refuse(f"positions is a contiguous int32 tensor of ({rows},) on {self.device}")
            pos_at = positions.data_ptr()
        else:
            if lens is None or lens.dtype is not self._i32 or lens.device != self.device or lens.dim() != 1 or not lens.is_contiguous():
                _refuse(f"lens is a contiguous int32 tensor (sequences,) on {self.device}")
            n, lens_at = len(lens), lens.data_ptr()
            if cu is not None:
                if cu.dtype is not self._i32 or cu.device != self.device or cu.dim() != 1 or len(cu) != n + 1 or not cu.is_contiguous():
                    _refuse("cu is a contiguous int32 tensor, with one entry more than there are sequences")
                cu_at = cu.data_ptr()
            elif rows != n:
                _refuse(f"without cu every sequence brings one row: got {rows} rows for {n} sequences")
        to_q, to_k = (None, None) if out is None else (out, None) if k is None else out
        q, out_q, x = self._rows(q, to_q, dtype, rows, "q")
        if k is None:
            status = self._rotate(c, self._get_stream(self._index), C.byref(x), 1, rows, lens_at, cu_at, n, pos_at, back)
        else:
            k, out_k, y = self._rows(k, to_k, dtype, rows, "k")
            if out is not None and x.out == y.out and rows:
                _refuse("the results of q and k are written to places that are apart from one another")
            status = self._rotate(c, self._get_stream(self._index), self._two(x, y), 2, rows, lens_at, cu_at, n, pos_at, back)
        if status:
            check(status)
        return out_q if k is None else (out_q, out_k)


__all__ = ["Rotary"]
