"""The 4-bit key/value cache on the CPU in 64 bits, from its definition: codes, scales and where they lie, and attention."""
import math

import torch

from tests.kv_plain import PlainCache

# every scale, ascending: multiples of 2^-17 up to 2^-14, then four significant bits
SCALES = torch.tensor([m * 2.0**-17 for m in range(8)] + [m * 2.0**e for e in range(-17, 14) for m in range(8, 16)], dtype=torch.float64)
SCALES = SCALES[SCALES <= 9216]


def coded4(x):
    """(codes from -7 to 7, numbers of the scales) of rows (..., dim) in float64; 255: no number."""
    y = x.unflatten(-1, (-1, 32))
    most = y.abs().amax(-1)
    fine = torch.isfinite(y).all(-1)
    # the smallest scale that is not below a seventh: 7 times a scale is exact
    n = torch.searchsorted(7 * SCALES, torch.where(fine, most, 0.0)).clamp(max=len(SCALES) - 1)
    s = torch.where(n > 0, SCALES[n], 1.0)[..., None]
    codes = torch.where(fine[..., None] & (n > 0)[..., None], (torch.where(fine[..., None], y, 0.0) / s).round().clamp(-7, 7), 0.0)
    return codes, torch.where(fine, n, 255)


def values4(codes, n):
    return (codes * torch.where(n == 255, math.nan, SCALES[n.clamp(max=len(SCALES) - 1)])[..., None]).flatten(-2)


def packed4(codes):
    """Bytes as the header describes them: of every 16 bits four neighbouring components, 16 bits u * groups + g from 32 g + 4 u on."""
    groups = codes.shape[-2]
    out = torch.zeros((*codes.shape[:-2], groups * 16), dtype=torch.int64)
    for g in range(groups):
        for c in range(32):
            at = (c // 4 * groups + g) * 4 + c % 4
            out[..., at // 2] |= (codes[..., g, c].long() + 8) << 4 * (at % 2)
    return out.to(torch.uint8)


class PlainFour(PlainCache):
    """k and v hold the values that the codes stand for, k_scale and v_scale the largest of a row's scales that is a number."""

    def __init__(self, pages, heads, dim, page_size, dtype):
        super().__init__(pages, heads, dim, page_size, dtype, "same")

    def hold(self, name, codes, n):
        """All rows of k or v."""
        getattr(self, name).copy_(values4(codes, n))
        getattr(self, name + "_scale").copy_(torch.where(n == 255, 0.0, SCALES[n.clamp(max=len(SCALES) - 1)]).amax(-1))

    def add(self, k, v, table, lens, cu=None):
        coded = [coded4(x.double()) for x in (k, v)]
        rounded, scale = [values4(*x) for x in coded], [torch.where(n == 255, 0.0, SCALES[n.clamp(max=len(SCALES) - 1)]).amax(-1) for _, n in coded]
        super().add(k, v, table, lens, cu)  # bounds are those of the rows as they came
        for r, b, pos in self.places(table, lens, cu):
            page = self.page(table, b, pos // self.page_size) if pos >= 0 else -1
            if page >= 0:
                slot = pos % self.page_size
                self.k[page, :, slot], self.v[page, :, slot] = rounded[0][r], rounded[1][r]
                self.k_scale[page, :, slot], self.v_scale[page, :, slot] = scale[0][r], scale[1][r]

    def attend(self, q, table, lens, cu, blocks, scale, out, lse):
        """As the plain cache's, with tolerances of its own; s is a row's largest scale.

        Scores: sums of exact products, of which the groups' are added up one by one: 8 steps more than in the plain cache.  bf16
        queries become fp16 relative to their largest component, and components lose at most 2^-38 of it.
        Weights: rounded to fp16, 2^-11 of themselves, and for results in bf16 once more as the product with a scale.  2^(7 - unit) stands for a weight of 1,
        where 2^unit is 1 or at most half the largest scale, and the step of the smallest numbers is 2^-24: each is off by 2^-32 max(1, s / 2),
        which meets 7 s, and its product by as much, which meets 7.  Values: n products in 32 bits."""
        group, half = q.shape[1] // self.heads, torch.finfo(self.dtype).eps / 2
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        for r, b, pos in self.places(table, lens, cu):
            for h in range(self.heads):
                sl = slice(h * group, (h + 1) * group)
                chosen, most = [], -1
                for e in range(pos // self.page_size + 1 if pos >= 0 else 0) if blocks is None else blocks[r, h].tolist():
                    if most < e < table.shape[1] and e * self.page_size <= pos:
                        chosen.append(e)
                        most = e
                at = [(self.page(table, b, j), j) for j in chosen]
                pages = torch.tensor([p for p, j in at if p >= 0 for s in range(min(self.page_size, pos + 1 - j * self.page_size))], dtype=torch.long)
                slots = torch.tensor([s for p, j in at if p >= 0 for s in range(min(self.page_size, pos + 1 - j * self.page_size))], dtype=torch.long)
                n = len(pages)
                if n == 0:
                    out[r, sl], lse[r, sl] = 0, -math.inf
                    continue
                k, v, x = self.k[pages, h, slots], self.v[pages, h, slots], q[r, sl].double()
                vs = self.v_scale[pages, h, slots]
                s = x @ k.T * scale
                off = abs(scale) * ((self.dim + 8) * 2.0**-24 * float((x.abs() @ k.abs().T).nan_to_num(posinf=0).max())
                                    + self.dim * 2.0**-38 * float(x.abs().max().nan_to_num(posinf=0) * k.abs().nan_to_num().max()))
                w = torch.exp(s - s.amax(-1, keepdim=True))
                w = torch.where(w < 2.0**-126, 0.0, w)
                p = w / w.sum(-1, keepdim=True)
                out[r, sl] = torch.where(p[..., None] > 0, p[..., None] * v, torch.where(p.isnan(), torch.nan, 0.0)[..., None]).sum(1)
                lse[r, sl] = torch.logsumexp(s, -1)
                weight = (2.0**-11 if self.dtype == torch.float16 else 2.0**-10) + 2 * off + 2 * n * 2.0**-24 + 2.0**-20
                tol[r, sl] = (p @ v.abs().nan_to_num()) * weight + out[r, sl].abs().nan_to_num(posinf=0) * half * 1.001
                tol[r, sl] += n * 2.0**-32 * max(1.0, float(vs.max()) / 2) * 7 * (float(vs.max()) + 1)
                tol[r, sl] += torch.finfo(self.dtype).smallest_normal * half
                ltol[r, sl] = off + n * 2.0**-24 + lse[r, sl].abs() * 2.0**-22 + 2.0**-20
        return out, lse, tol, ltol
