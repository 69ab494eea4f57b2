"""Attention of single rows over 4 bits whose values are small, or of very different sizes: results are as near as their values allow."""
import math

import pytest
import torch

from tests.kv_plain_four import SCALES, packed4
from tests.test_gpu_kv_rows import batch, i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
SMALL = {"multiples of 2^-17": (1, 8), "2^-14 to 2^-12": (8, 24), "2^-12 to 2^-7": (24, 64), "2^-5 to 2": (80, 128)}


def cache(lens, heads, group, dim, page, dtype, sizes, seed=0):
    """A cache whose keys have scores within one of each other but for one in every sequence, 10 or 11 above them, whose values are
    zero; the others' values are of one sign, with scales sizes(n rows).  (cache, queries, table, keys, values and
    values' scales of each sequence)"""
    import ferrolm_b200 as fv

    g = torch.Generator().manual_seed(seed)
    blocks = -(-max(lens) // page) + 1
    c = fv.KvCache(len(lens) * blocks + 3, heads, dim, page_size=page, dtype=dtype, kind="int4x32")
    for name in ("k_scale", "v_scale"):  # what nobody sees: the largest, and no numbers
        x = getattr(c, name)
        x.copy_(torch.tensor([225, 255], dtype=torch.uint8)[torch.randint(0, 2, x.shape, generator=g)])
    table = batch(len(lens), blocks, c.pages, seed + 1)
    base = torch.randn((heads, 1, dim), generator=g)
    q = (base + 0.02 * torch.randn((len(lens), heads, group, dim), generator=g)).reshape(len(lens), heads * group, dim).to(dtype)
    keys, values, scales_of = [], [], []
    for b, n in enumerate(lens):
        kc, vc = torch.randint(-7, 8, (n, heads, dim // 32, 32), generator=g).double(), torch.randint(1, 8, (n, heads, dim // 32, 32), generator=g).double()
        kn, vn = torch.full((n, heads, dim // 32), 72), sizes(n, g)[:, None, None].expand(n, heads, dim // 32).clone()
        if n:
            far = n // 3
            kc[far], vc[far] = 7 * base.view(heads, dim // 32, 32).sign(), 0
            score = (base.abs().sum(-1) * 7 * dim**-0.5).view(heads, 1)  # of a scale of 1
            kn[far] = torch.searchsorted(SCALES, 10.5 / score.double())
            at = table[b, torch.arange(n) // page].long(), torch.arange(n) % page
            for held, scales, codes, m in ((c.k, c.k_scale, kc, kn), (c.v, c.v_scale, vc, vn)):
                y = held.cpu()
                y[at[0], :, at[1]] = packed4(codes)
                held.copy_(y)
                y = scales.cpu()
                y[at[0], :, at[1]] = m.to(torch.uint8)
                scales.copy_(y)
        keys.append((kc * SCALES[kn][..., None]).flatten(-2)), values.append((vc * SCALES[vn][..., None]).flatten(-2)), scales_of.append(SCALES[vn])
    return c, q, table, keys, values, scales_of


def check(got, lse, q, keys, values, scales, dtype):
    """Against 64 bits.  Scores: dim exact products and 8 steps of sums in 32 bits, queries that become fp16 lose 2^-38 of the largest.  Weights:
    rounded to fp16 once, 2^-11, but by no less than the smallest fp16 allows, 2^-32 of the largest weight.  Values are exact, at most 7 scales.
    Sums of n in 32 bits; the result is rounded once."""
    heads, dim = keys[0].shape[1], keys[0].shape[2]
    group = q.shape[1] // heads
    for b, (k, v) in enumerate(zip(keys, values)):
        n = len(k)
        for h in range(heads):
            sl = slice(h * group, (h + 1) * group)
            y, z = got[b, sl].cpu().double(), lse[b, sl].cpu().double()
            if n == 0:
                assert (y == 0).all() and (z == -math.inf).all()
                continue
            x = q[b, sl].double()
            s = x @ k[:, h].T * dim**-0.5
            off = dim**-0.5 * ((dim + 8) * 2.0**-24 * float((x.abs() @ k[:, h].abs().T).max()) + dim * 2.0**-38 * float(x.abs().max() * k[:, h].abs().max()))
            w = torch.exp(s - s.amax(-1, keepdim=True))
            total = w.sum(-1, keepdim=True)
            want = w / total @ v[:, h]
            most = float(scales[b][:, h].max())
            tol = (w / total @ v[:, h].abs()) * (2.0**-11 * 1.001 + 2 * off + 2 * n * 2.0**-24 + 2.0**-20)
            tol += 7 * n / total * 2.0**-32 * most
            tol += want.abs() * torch.finfo(dtype).eps / 2 * 1.001 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
            assert ((y - want).abs() <= tol).all(), (b, h, float(((y - want).abs() / want.abs()).max()), float((tol / want.abs()).max()))
            assert ((z - torch.logsumexp(s, -1)).abs() <= off + n * 2.0**-24 + 2.0**-18).all()


@pytest.mark.parametrize("size", list(SMALL))
@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 1, 4, 128, 64), (BF, 2, 3, 96, 16), (BF, 1, 12, 64, 32), (BF, 1, 20, 96, 128), (FP, 1, 5, 128, 32)])
@pytest.mark.parametrize("lens", [[6001], [2500, 17, 0, 1, 900]])
def test_values_of_one_size(size, dtype, heads, group, dim, page, lens):
    """Most of the result comes from thousands of rows that weigh 2^-15 each."""
    lo, hi = SMALL[size]
    c, q, table, *held = cache(lens, heads, group, dim, page, dtype, lambda n, g: torch.randint(lo, hi, (n,), generator=g))
    at = q.cuda(), table.cuda(), i32(lens).cuda()
    got, lse = c.attend(*at, return_lse=True)
    check(got, lse, q, *held, dtype)
    # a list of all blocks is the same, and a CTA for each task, without a place to share the work out in, as near
    every = torch.arange(table.shape[1], dtype=torch.int32).expand(len(lens), heads, -1).contiguous().cuda()
    check(*c.attend(*at, blocks=every, return_lse=True), q, *held, dtype)
    b, out = c._batch(at[1], at[2], None, len(lens)), torch.zeros_like(got)
    import ferrolm_b200 as fv

    fv.kv.check(c._attend(c._ref, torch.cuda.current_stream().cuda_stream, b, at[0].data_ptr(), at[0].stride(0), at[0].stride(1), group, None, 0, dim**-0.5, out.data_ptr(), lse.data_ptr(), None, 0))
    check(out, lse, q, *held, dtype)


@pytest.mark.parametrize("order", ["up", "down", "one in the middle"])
@pytest.mark.parametrize("low,high", [(2, 30), (8, 100), (20, 160), (100, 225)])
@pytest.mark.parametrize("dtype,group,dim", [(BF, 4, 128), (BF, 9, 96), (FP, 2, 64)])
def test_values_that_grow(order, low, high, dtype, group, dim):
    """Small scales before large ones and behind them, and a single row far above the others."""

    def sizes(n, g):
        x = torch.linspace(low, high, n).round().long()
        return x if order == "up" else x.flip(0) if order == "down" else torch.where(torch.arange(n) == n // 2, high, low)

    lens = [3011, 700]
    c, q, table, *held = cache(lens, 1, group, dim, 32, dtype, sizes)
    check(*c.attend(q.cuda(), table.cuda(), i32(lens).cuda(), return_lse=True), q, *held, dtype)


@pytest.mark.parametrize("size", list(SMALL))
def test_single_rows_are_as_prompts(size):
    """The last rows of a sequence, by themselves and as a prompt: weights that are rounded by 2^-11 each, and two results in bf16,
    whose half step is eps / 2 = 2^-8 of the value."""
    lo, hi = SMALL[size]
    c, q, table, *held = cache([5000], 2, 4, 128, 64, BF, lambda n, g: torch.randint(lo, hi, (n,), generator=g))
    x, at = q.cuda().expand(6, -1, -1).contiguous(), (table.cuda(), i32([5000]).cuda())
    prompt = c.attend(x, *at, cu=i32([0, 6]).cuda())[5].float()
    alone = c.attend(x[5:], *at)[0].float()
    assert ((prompt - alone).abs() <= prompt.abs() * (2 * 2.0**-11 + 2 * 2.0**-8 + 2.0**-12)).all()
