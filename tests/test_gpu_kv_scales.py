"""KvCache.attend of prompts over 8 bits where the rows' scales are many powers of two apart: what a query does not see has no part
in its result, whichever queries share its tile."""
import math

import pytest
import torch

from tests.test_gpu_kv_attend import check, lists, pair, queries
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def put(c, p, page, slot, scale):
    for y in (c, p):
        y.v_scale[page, :, slot] = scale


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("power", [26, 45, 100])
def test_rows_that_only_other_queries_see(kind, dtype, page, power):
    """A value's scale 2^26 to 2^100 times the others': behind the position of half of a prompt's rows, or in a block that only some of
    them list.  The others' results are those that they have without it, to the bit, and right."""
    heads, group, dim, new = 2, 4, 64, 40
    c, p = pair(14, heads, dim, page, dtype, kind, seed=power)
    table = i32([[4, 2, 7, 1, 0, 5, 9, 3, 12, 6]])
    n = 9 * page + 11
    q, cu = queries(new, heads, group, dim, dtype, 2), i32([0, new])

    def both(blocks, lens, far, seen, page_at, slot):
        plain = float(c.v_scale[page_at, 0, slot])
        before = check(c, p, q, table, lens, cu, blocks)
        put(c, p, page_at, slot, far)
        after = check(c, p, q, table, lens, cu, blocks)
        assert (~seen).any() and seen.any()
        for x, y in zip(before, after):
            assert torch.equal(x[~seen], y[~seen])
        put(c, p, page_at, slot, plain)

    # the row at the position of the call's 20th: the first 20 do not see it
    at = n - new + 20
    both(None, [n], 2.0**power, torch.arange(new) >= 20, int(table[0, at // page]), at % page)
    # block 3, which every third row lists
    blocks = lists(new, heads, 5, 9, 3)
    seen = torch.arange(new) % 3 == 0
    for r in range(new):
        for h in range(heads):
            x = [b for b in blocks[r, h].tolist() if b not in (-1, 3)][:4]
            x = sorted(x + [3] if seen[r] else x)
            blocks[r, h] = i32(x + [-1] * (5 - len(x)))
    both(blocks, [n], 2.0**power, seen, int(table[0, 3]), 5)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("low,high", [(-14, 6), (-40, -20), (-149, -120), (-3, 3)])
def test_scales_that_rise_and_fall_along_a_prompt(kind, dtype, page, low, high):
    """Scales of the values that grow or shrink by many powers of two, down to those that have no whole exponent, zeros among them:
    every query's power of two follows what it sees, by position and by lists."""
    heads, group, dim, new = 1, 6, 96, 50
    c, p = pair(12, heads, dim, page, dtype, kind, seed=high)
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(12, generator=g)[:8].view(1, 8).to(torch.int32)
    q, cu, n = queries(new, heads, group, dim, dtype, 1), i32([0, new]), 8 * page - 5
    q[3] *= 64
    q[4] /= 4096
    q[5] = 0
    for order in (1, -1):
        scale = torch.exp2((torch.linspace(low, high, 8 * page, dtype=torch.float64) * order + (low + high if order < 0 else 0))) * torch.rand(8 * page, generator=g)
        scale[3 * page + 4 : 3 * page + 9] = 0
        c.v_scale.zero_()
        c.v_scale[table[0].long(), 0] = scale.float().view(8, page).cuda()
        p.v_scale.copy_(c.v_scale.cpu().double())
        check(c, p, q, table, [n], cu, None)
        check(c, p, q, table, [n], cu, lists(new, heads, 4, 8, 5))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
def test_a_value_that_is_no_number_beside_scales_far_apart(kind, page):
    """NaN for the queries that see the row, and for the others what they have without it, to the bit."""
    heads, group, dim, new, dtype = 2, 2, 128, 70, BF
    c, p = pair(9, heads, dim, page, dtype, kind)
    table, n = i32([[4, 2, 7, 1, 0, 5, 3]]), 6 * page + 9
    put(c, p, 7, 2, 2.0**50)
    q, cu = queries(new, heads, group, dim, dtype, 2), i32([0, new])
    at = n - new + 33
    where, slot = int(table[0, at // page]), at % page
    for b in (None, lists(new, heads, 5, 6, 3)):
        before = check(c, p, q, table, [n], cu, b)
        kept = c.v_scale.clone()
        put(c, p, where, slot, torch.nan)
        after = c.attend(q.cuda(), table.cuda(), i32([n]).cuda(), cu=cu.cuda(), blocks=None if b is None else b.cuda()).cpu()
        sees = (torch.arange(new) >= 33)[:, None].expand(new, heads)
        if b is not None:
            sees = sees & (b == at // page).any(-1)
        sees = sees.repeat_interleave(group, 1)
        assert torch.equal(after[~sees], before[0].cpu()[~sees]) and not after[~sees].isnan().any() and sees.any()
        for r, h in sees.nonzero().tolist():
            # A weight is held as 2^14 of it, down to 2^-126: from 2^-140 on, and with a score's error of far less than 14 surely from 2^-126
            # on, it carries the NaN; below, it may be none, and no weight carries nothing.
            seen = torch.tensor([i for i in range(n - new + r + 1) if b is None or i // page in b[r, h // group].tolist()])
            rows = table[0, seen // page].long()
            keys = p.k[rows, h // group, seen % page] * p.k_scale[rows, h // group, seen % page][:, None]
            score = keys @ q[r, h].double() * dim**-0.5
            weight = float(score[seen == at] - score.max()) / math.log(2)
            assert after[r, h].isnan().all() if weight >= -126 else after[r, h].isnan().all() or not after[r, h].isnan().any(), (r, h, weight)
        c.v_scale.copy_(kept)
        p.v_scale.copy_(kept.cpu().double())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("low,high", [(-40, -20), (-149, -120), (-30, 10)])
@pytest.mark.parametrize("blocks", [5, 70])
def test_scales_that_rise_and_fall_before_single_rows(kind, dtype, low, high, blocks):
    """The same for rows by themselves, by a CTA each and in parts."""
    heads, group, dim, page, B = 1, 5, 128, 16, 3
    c, p = pair(B * blocks, heads, dim, page, dtype, kind, seed=high)
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32)
    lens = [blocks * page, blocks * page - 7, 3 * page + 1]
    q = queries(B, heads, group, dim, dtype, 1)
    for order in (1, -1):
        scale = torch.exp2(torch.linspace(low, high, blocks * page, dtype=torch.float64) * order + (low + high if order < 0 else 0)) * torch.rand((B, blocks * page), generator=g)
        scale[:, 2 * page + 4 : 2 * page + 9] = 0
        c.v_scale[table.long().flatten(), 0] = scale.float().view(B * blocks, page).cuda()
        p.v_scale.copy_(c.v_scale.cpu().double())
        check(c, p, q, table, lens, None, None)
        check(c, p, q, table, lens, None, lists(B, heads, 4, 5, 5))
