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

    def attend(self, q, table, lens, cu, blocks, scale, out, lse):
        """Into the given float64 tensors, and how far a result may be off: (out, lse, out's tolerance, lse's tolerance).

        A score of dim products summed in 32 bits, then multiplied three times, is off by at most (dim + 4) 2^-24 times the sum
        of the products' absolute values; a weight by that of its own and of the largest score (all are relative to it), by
        2^-11 for its rounding to 16 bits (2^-8 where `out`'s type is bf16 and the rows are a prompt's), by 2^-20 for 2^x and
        the factors that join parts; a sum of n terms in 32 bits by n 2^-24 of the sum of absolute values, and so is the sum
        of weights.  All of it scales sum |p v|; on top comes the result's own rounding.  A weight in fp16, where 2^14 stands
        for 1 and the step of the smallest numbers is 2^-24, is off by up to 2^-25 / 2^14 = 2^-39 however small it is; it is
        held relative to a power of two of at most twice the largest scale, and the sum of weights is at least 1: n rows add
        n 2^-38 times the largest scale times the largest code."""
        group, half = q.shape[1] // self.heads, torch.finfo(self.dtype).eps / 2
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        for r, b, pos in self.places(table, lens, cu):
            for h in range(self.heads):
                if blocks is None:
                    chosen = range(pos // self.page_size + 1 if pos >= 0 else 0)
                else:
                    chosen, most = [], -1
                    for e in blocks[r, h].tolist():
                        if most < e < table.shape[1] and e * self.page_size <= pos:
                            chosen.append(e)
                            most = e
                at = [(self.page(table, b, j), j) for j in chosen]
                rows = [(p, j * self.page_size + s, s) for p, j in at if p >= 0 for s in range(self.page_size) if j * self.page_size + s <= pos]
                sl = slice(h * group, (h + 1) * group)
                if not rows:
                    out[r, sl], lse[r, sl] = 0, -math.inf
                    continue
                pages, slots = torch.tensor([x[0] for x in rows]), torch.tensor([x[2] for x in rows])
                k, v = self.k[pages, h, slots], self.v[pages, h, slots]
                if self.kind != "same":
                    k, v = k * self.k_scale[pages, h, slots][:, None], v * self.v_scale[pages, h, slots][:, None]
                x = q[r, sl].double()
                s = x @ k.T * scale
                off = (self.dim + 4) * 2.0**-24 * float((x.abs() @ k.abs().T).nan_to_num(posinf=0).max()) * abs(scale)
                w = torch.exp(s - s.amax(-1, keepdim=True))
                w = torch.where(w < 2.0**-126, 0.0, w)  # the smallest power of two in 32 bits: what is below has no weight
                p = w / w.sum(-1, keepdim=True)
                out[r, sl] = torch.where(p[..., None] > 0, p[..., None] * v, torch.where(p.isnan(), torch.nan, 0.0)[..., None]).sum(1)
                lse[r, sl] = torch.logsumexp(s, -1)
                n = len(rows)
                floor = self.v[pages, h, slots].nan_to_num(posinf=0, neginf=0).abs().max() * (1 if self.kind == "same" else self.v_scale[pages, h, slots].nan_to_num().max())
                weight = (2.0**-8 if self.dtype == torch.bfloat16 and self.kind == "same" else 2.0**-11) + 2 * off + 2 * n * 2.0**-24 + 2.0**-20
                tol[r, sl] = (p @ v.abs().nan_to_num(posinf=0)) * weight + out[r, sl].abs().nan_to_num(posinf=0) * half * 1.001 + n * 2.0**-38 * floor + torch.finfo(self.dtype).smallest_normal * half
                ltol[r, sl] = off + n * 2.0**-24 + lse[r, sl].abs() * 2.0**-22 + 2.0**-20
        return out, lse, tol, ltol
