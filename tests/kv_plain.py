"""A key/value cache on the CPU in 64 bits, row by row from the definitions: what the kernels' tests compare with."""
import math

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}


def coded(x, kind):
    """(codes, scale) of a row (float64).  The quotient in 64 bits is off by 2^-53 of itself, and one of two values of at
    most 11 bits that is not a border of two codes is further from it than 2^-13: rounding it gives the true code."""
    top, most = TOP[kind], x.abs().max()
    if not torch.isfinite(most):
        return torch.zeros_like(x), math.nan
    y = x * top / most if most > 0 else torch.zeros_like(x)
    y = y.round() if kind == "int8" else y.to(torch.float32).to(torch.float8_e4m3fn).double()
    return y, float((most.float() / torch.tensor(top, dtype=torch.float32)))


class PlainCache:
    def __init__(self, pages, heads, dim, page_size, dtype, kind):
        self.pages, self.heads, self.dim, self.page_size, self.dtype, self.kind = pages, heads, dim, page_size, dtype, kind
        z = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
        self.k, self.v = z(pages, heads, page_size, dim), z(pages, heads, page_size, dim)
        self.k_scale, self.v_scale = z(pages, heads, page_size), z(pages, heads, page_size)
        self.bounds, self.bound_codes, self.bound_scale = z(pages, heads, 2, dim), z(pages, heads, 2, dim), z(pages, heads)

    def page(self, table, b, j):
        if not 0 <= j < table.shape[1]:
            return -1
        p = int(table[b, j])
        return p if 0 <= p < self.pages else -1

    def places(self, table, lens, cu):
        """(row of the call, sequence, position) of every row that belongs to a sequence."""
        cu = list(range(table.shape[0] + 1)) if cu is None else [int(x) for x in cu]
        for b in range(table.shape[0]):
            n = cu[b + 1] - cu[b]
            for i in range(n):
                yield cu[b] + i, b, int(lens[b]) - n + i

    def add(self, k, v, table, lens, cu=None):
        touched = {}
        for r, b, pos in self.places(table, lens, cu):
            page = self.page(table, b, pos // self.page_size) if pos >= 0 else -1
            if page < 0:
                continue
            slot = pos % self.page_size
            for h in range(self.heads):
                for x, to, scales in ((k, self.k, self.k_scale), (v, self.v, self.v_scale)):
                    row = x[r, h].double()
                    if self.kind == "same":
                        to[page, h, slot] = row
                    else:
                        to[page, h, slot], scales[page, h, slot] = coded(row, self.kind)
                row = torch.where(torch.isfinite(k[r, h]), k[r, h], 0).double()
                fresh = slot == 0
                self.bounds[page, h, 0] = row if fresh else torch.minimum(self.bounds[page, h, 0], row)
                self.bounds[page, h, 1] = row if fresh else torch.maximum(self.bounds[page, h, 1], row)
                touched[page, h] = True
        for page, h in touched:
            codes, scale = coded(self.bounds[page, h].flatten(), "int8")
            self.bound_codes[page, h], self.bound_scale[page, h] = codes.view(2, -1), scale

    def value(self, name, page, h, slot):
        x = getattr(self, name)[page, h, slot]
        return x if self.kind == "same" else x * getattr(self, name + "_scale")[page, h, slot]

    def vectors(self, table, lens, cu, out_k, out_v):
        """Into the given float64 tensors; the product of a code and a scale has at most 32 bits, so it is rounded to 32 bits
        and then to the cache's type exactly as the definition has it."""
        for r, b, pos in self.places(table, lens, cu):
            page = self.page(table, b, pos // self.page_size) if pos >= 0 else -1
            if page >= 0:
                for name, out in (("k", out_k), ("v", out_v)):
                    for h in range(self.heads):
                        out[r, h] = self.value(name, page, h, pos % self.page_size).float().to(self.dtype).double()
        return out_k, out_v

    def search(self, q, table, lens, k, cu, first, recent, out):
        """Into the given int64 tensor.  Sums of whole numbers in 64 bits; the score has the definition's two roundings to 32."""
        group = q.shape[1] // self.heads
        for r, b, pos in self.places(table, lens, cu):
            for h in range(self.heads):
                x = q[r, h * group : (h + 1) * group]
                x = torch.where(torch.isfinite(x), x, 0).double()
                codes = coded(x.flatten(), "int8")[0].view(group, -1)
                parts = torch.cat((codes.clamp(max=0).sum(0), codes.clamp(min=0).sum(0)))
                parts = (parts * 127.0 / parts.abs().max().clamp(min=1)).round()
                last, scored = pos // self.page_size if pos >= 0 else -1, []
                for j in range(last + 1):
                    page = self.page(table, b, j)
                    if page < 0:
                        continue
                    s = (parts * self.bound_codes[page, h].flatten()).sum().float() * self.bound_scale[page, h].float()
                    forced = j < first or j > last - recent
                    scored.append((-math.inf if forced else -float(s), j))
                chosen = sorted(j for _, j in sorted(scored)[:k])
                out[r, h] = torch.tensor(chosen + [-1] * (k - len(chosen)))
        return out
