"""KvCache.search_blocks against scores that nothing is rounded in: a block that is left out promises no more than one that is taken,
but for what the roundings of queries and bounds to 8 bits may come to."""
import pytest
import torch

from tests.kv_plain import coded
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def unrounded(q, lo, hi, group):
    """Sums over a group's heads of the largest inner products that the bounds allow, and how far the scores are from them.

    q (group, dim), lo and hi (blocks, dim), all in 64 bits.  With a = max|q| / 127 a query's component is off by a / 2 and the sum of a
    group's positive (or negative) ones by group a / 2; these sums are rounded again, to 127 steps of the largest, M a: by M a / 254.  A
    bound is off by half of its block's b = max(|lo|, |hi|) / 127.  |x y - X Y| <= |x - X| |y| + |X| |y - Y| for each of the 2 dim
    products.  A sum of whole numbers is exact; its product with the block's scale has two roundings to 32 bits."""
    plus, minus = q.clamp(min=0).sum(0), q.clamp(max=0).sum(0)
    exact = hi @ plus + lo @ minus
    codes = coded(q.flatten(), "int8")[0].view(group, -1)
    a = float(q.abs().max()) / 127
    most = float(torch.maximum(codes.clamp(min=0).sum(0).max(), (-codes.clamp(max=0)).sum(0).max()))
    off = a * (group / 2 + most / 254)  # of a sum over the group
    b = torch.maximum(lo.abs(), hi.abs()).amax(-1) / 127
    size = lo.abs().sum(-1) + hi.abs().sum(-1)
    sums = plus.abs().sum() + minus.abs().sum() + 2 * q.shape[1] * off  # of the rounded ones, at most
    error = off * size + sums * b / 2
    return exact, error + (exact.abs() + error) * 2.0**-22


@pytest.mark.parametrize("dtype,heads,group,dim,page,new", [(BF, 2, 4, 128, 32, 1), (FP, 2, 7, 96, 16, 1), (BF, 1, 16, 64, 64, 24), (FP, 1, 1, 128, 16, 40)])
@pytest.mark.parametrize("spread", [0.0, 2.0, 6.0])
def test_what_is_left_out_promises_no_more(dtype, heads, group, dim, page, new, spread):
    """Query heads of one size, of sizes a few times and hundreds of times apart (the small ones round to nothing, and weigh as
    little in the sum); keys with channels that stand out."""
    import ferrolm_b200 as fv

    blocks, k, first, recent = 60, 9, 1, 2
    g = torch.Generator().manual_seed(int(spread) + dim)
    c = fv.KvCache(blocks, heads, dim, page_size=page, dtype=dtype)
    n = blocks * page - 3
    table = torch.randperm(blocks, generator=g).view(1, blocks).to(torch.int32)
    keys = torch.randn((n, heads, dim), generator=g) * 0.5 + torch.randn((blocks, heads, dim), generator=g).repeat_interleave(page, 0)[:n]
    keys[:, :, ::11] += 4
    keys = keys.to(dtype)
    c.add(keys.cuda(), keys.cuda(), table.cuda(), i32([n]).cuda(), cu=i32([0, n]).cuda())
    q = (torch.randn((new, heads * group, dim), generator=g) * torch.exp(spread * torch.randn((new, heads * group, 1), generator=g))).clamp(-1000, 1000).to(dtype)
    got = c.search_blocks(q.cuda(), table.cuda(), i32([n]).cuda(), k, cu=i32([0, new]).cuda(), first=first, recent=recent).cpu().long()
    left_out = 0
    for r in range(new):
        last = (n - new + r) // page
        for h in range(heads):
            taken = got[r, h].tolist()
            assert len(set(taken)) == k and taken == sorted(taken) and set(range(first)) | set(range(last - recent + 1, last + 1)) <= set(taken)
            rows = keys[: n - new + r + 1, h].double()  # the last block's bounds hold the call's later rows too, but it is taken anyhow
            lo = torch.stack([rows[j * page : (j + 1) * page].amin(0) for j in range(last + 1)])
            hi = torch.stack([rows[j * page : (j + 1) * page].amax(0) for j in range(last + 1)])
            exact, error = unrounded(q[r, h * group : (h + 1) * group].double(), lo, hi, group)
            free = [j for j in taken if first <= j <= last - recent]
            others = [j for j in range(first, last - recent + 1) if j not in taken]
            assert (exact[free][:, None] + error[free][:, None] >= exact[others][None] - error[others][None]).all(), (r, h)
            best = sorted(range(first, last - recent + 1), key=lambda j: -float(exact[j]))[: len(free)]
            left_out += len(set(best) - set(free))
    print(f"{left_out} of {new * heads * (k - first - recent)} blocks are others than without rounding")
