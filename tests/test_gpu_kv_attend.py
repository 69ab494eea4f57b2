"""KvCache.attend against the cache of tests/kv_plain.py, whose attend() says how far a result may be off and why."""
import pytest
import torch

from tests.kv_plain import PlainCache
from tests.test_gpu_kv_rows import batch, cuda, i32, rows

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def pair(pages, heads, dim, page, dtype, kind, seed=0):
    """Caches with random rows; channels that stand out, rows of unequal size."""
    import ferrolm_b200 as fv

    g = torch.Generator().manual_seed(seed)
    c, p = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind=kind), PlainCache(pages, heads, dim, page, dtype, kind)
    for name in ("k", "v"):
        x = torch.randn((pages, heads, page, dim), generator=g)
        x[..., ::9] *= 3
        if kind == "same":
            x = x.to(dtype)
            getattr(c, name).copy_(x)
            getattr(p, name).copy_(x)
        else:
            codes = (x * 30).clamp(-127, 127).round() if kind == "int8" else (x * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
            scale = torch.exp(torch.randn((pages, heads, page), generator=g)) / (30 if kind == "int8" else 60)
            getattr(c, name).copy_(codes.to(getattr(c, name).dtype))
            getattr(c, name + "_scale").copy_(scale)
            getattr(p, name).copy_(codes.double())
            getattr(p, name + "_scale").copy_(scale)
    return c, p


def queries(n, heads, group, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((n, heads * group, dim), generator=g) * torch.exp(0.7 * torch.randn((n, heads * group, 1), generator=g))).to(dtype)


def lists(n, heads, k, most, seed):
    """Ascending lists of blocks, some short, some with entries that are to be skipped."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((n, heads, k), -1, dtype=torch.int32)
    for r in range(n):
        for h in range(heads):
            x = torch.randperm(max(most, 1), generator=g)[: int(torch.randint(0, k + 1, (1,), generator=g))].sort().values
            out[r, h, : len(x)] = x.to(torch.int32)
    return out


def check(c, p, q, table, lens, cu, blocks, scale=None):
    kind = torch.full(q.shape, 7.5, dtype=q.dtype), torch.full(q.shape[:2], 7.5)
    got = c.attend(q.cuda(), table.cuda(), i32(lens).cuda(), cu=cuda(cu), blocks=cuda(blocks), scale=scale, return_lse=True,
                   out=tuple(x.cuda() for x in kind))
    want = p.attend(q, table, lens, cu, blocks, q.shape[2] ** -0.5 if scale is None else scale, kind[0].double(), kind[1].double())
    for x, y, tol in zip(got, want, want[2:]):
        x = x.cpu().double()
        # to nearest, a result from half a step above the type's largest number on is infinite
        largest = torch.finfo(q.dtype).max * (1 + torch.finfo(q.dtype).eps / 4)
        same = (x == y) | (x.isnan() & y.isnan()) | (x.isinf() & (x.sign() == y.sign()) & (y.abs() + tol >= largest))
        off = torch.where(same, 0.0, (x - y).abs())
        assert (same | (off <= tol)).all(), (float((off - tol).max()), (off > tol).nonzero()[:5].tolist(), x[off > tol][:5], y[off > tol][:5], tol[off > tol][:5])
    return got


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 3, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 2, 1, 128, 32), (BF, 1, 37, 96, 16), (FP, 1, 8, 64, 16)])
def test_tokens(kind, dtype, heads, group, dim, page):
    """A row for every sequence: no rows at all, one, a border's neighbours, and enough for several warps and CTAs."""
    lens = [0, 1, 15, 16, 17, page, page + 1, 9 * page - 3, 30 * page]
    c, p = pair(300, heads, dim, page, dtype, kind)
    table = batch(len(lens), 30, 300, 2)
    q = queries(len(lens), heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, None, None)
    check(c, p, q, table, lens, None, lists(len(lens), heads, 11, 30, 4), scale=0.21)


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("B,blocks", [(1, 40), (1, 9), (3, 130), (40, 3)])
def test_few_and_many_rows(kind, B, blocks):
    """Every number of CTAs to a row."""
    heads, group, dim, page, dtype = 2, 5, 128, 32, BF
    c, p = pair(B * blocks + 3, heads, dim, page, dtype, kind, seed=B)
    table = batch(B, blocks, c.pages, 2)
    lens = [blocks * page - 7 * b % (blocks * page) for b in range(B)]
    q = queries(B, heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, None, None)
    check(c, p, q, table, lens, None, lists(B, heads, 70, blocks, 5))


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 1, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 2, 1, 128, 32), (BF, 1, 37, 96, 16), (FP, 1, 3, 64, 32)])
def test_prompts(kind, dtype, heads, group, dim, page):
    """Ragged pieces of prompts, one from the first row on, one that brings more rows than its sequence has, one of no rows, and
    rows behind the last sequence; all blocks, lists of a few, and lists that have nothing in common."""
    news, lens = [40, 0, 13, 9, 25], [40, 5, 13 * page - 3, 6, 200]
    c, p = pair(120, heads, dim, page, dtype, kind)
    table = batch(5, 20, 120, 2)
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = int(cu[-1]) + 6
    q = queries(n, heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, cu, None)
    check(c, p, q, table, lens, cu, lists(n, heads, 7, 13, 4), scale=0.17)
    check(c, p, q, table, lens, cu, lists(n, heads, 3, 13, 5))
    check(c, p, q, table[:, :2], lens, cu, None)  # rows behind the table's last column


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_prompts_over_values_that_are_not_finite(kind, dtype):
    """NaN and infinities in rows that some of the rows of a tile see and others do not, by position and by their lists."""
    heads, group, dim, page = 1, 4, 64, 16
    c, p = pair(9, heads, dim, page, dtype, kind)
    table, n, new = i32([[4, 2, 7, 1, 0, 5]]), 6 * page - 2, 40
    for i, (at, s) in enumerate([(5, 3), (5, 9), (0, 15), (7, 2), (1, 0)]):
        x = [torch.nan, torch.inf, -torch.inf][i % 3]
        for y in (c, p):
            if kind == "same":
                y.v[at, 0, s, 3 + 5 * i] = x
            else:
                y.v_scale[at, 0, s] = torch.nan
                y.v[at, 0, s] = 0
    q, cu = queries(new, heads, group, dim, dtype, 2), i32([0, new])
    check(c, p, q, table, [n], cu, None)
    check(c, p, q, table, [n], cu, lists(new, heads, 4, 6, 3))


@pytest.mark.parametrize("kind", ["same", "e4m3"])
def test_lists_of_prompts_are_read_as_they_are_documented(kind):
    heads, group, dim, page, dtype = 1, 3, 64, 16, FP
    c, p = pair(12, heads, dim, page, dtype, kind)
    table = i32([[3, -1, 5, 7, 1, 0]])
    odd = [[0, 0, 0, 2], [5, 4, 3, 2], [2, 1, 3, 3], [-1, 7, 1, 2], [-5, 6, 2**31 - 1, 0], [-1, -1, -1, -1], [1, 1, 1, 1], [4, 5, 6, 7], [100, 2, 101, 3]]
    check(c, p, queries(9, heads, group, dim, dtype, 1), table, [6 * page], i32([0, 9]), i32([[x] for x in odd]))
    check(c, p, queries(9, heads, group, dim, dtype, 1), table, [3 * page + 4], i32([0, 9]), i32([[x] for x in odd]))


def test_rows_of_a_prompt_are_those_of_tokens():
    """A piece of a prompt at once and row by row, over lists of its own and over everything."""
    heads, group, dim, page, dtype = 4, 4, 128, 64, BF
    c, p = pair(300, heads, dim, page, dtype, "same", seed=5)
    table, n, new = batch(1, 60, 300, 1), 60 * page - 9, 70
    q = queries(new, heads, group, dim, dtype, 2)
    blocks = c.search_blocks(q.cuda(), table.cuda(), i32([n]).cuda(), 12, cu=i32([0, new]).cuda())
    for b in (blocks, None):
        whole = c.attend(q.cuda(), table.cuda(), i32([n]).cuda(), cu=i32([0, new]).cuda(), blocks=b)
        each = torch.cat([c.attend(q[i : i + 1].cuda(), table.cuda(), i32([n - new + 1 + i]).cuda(), blocks=None if b is None else b[i : i + 1]) for i in range(new)])
        # weights in bf16 on one side and in two parts on the other, then both results rounded: four halves of a step of the largest value
        assert (whole.float() - each.float()).abs().max() <= 4 * 2.0**-8 * each.float().abs().max()


@pytest.mark.parametrize("kind", ["same", "e4m3"])
def test_lists_are_read_as_they_are_documented(kind):
    """Twice the same block, descending ones, blocks behind the query or the table, negative numbers, pages that are none."""
    heads, group, dim, page, dtype = 1, 3, 64, 16, FP
    c, p = pair(12, heads, dim, page, dtype, kind)
    table = i32([[3, -1, 5, 7, 1, 0], [1, 2, 12, 2**31 - 1, 4, 6], [9, 8, 10, 11, -(2**31), 2]])
    lens = [6 * page, 5 * page + 3, 3 * page]
    q = queries(3, heads, group, dim, dtype, 1)
    for row in ([0, 0, 0, 2], [5, 4, 3, 2], [2, 1, 3, 3], [-1, 7, 1, 2], [-5, 6, 2**31 - 1, 0], [-1, -1, -1, -1], [1, 1, 1, 1], [4, 5, 6, 7], [100, 2, 101, 3]):
        check(c, p, q, table, lens, None, i32([[row]] * 3))
    check(c, p, q, table, lens, None, None)
    check(c, p, q, table[:, :4], lens, None, None)  # rows behind the table's last column
    check(c, p, q, table[:, :0], lens, None, None)  # no column at all


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 3])
def test_what_is_masked_is_not_read_into_results(kind, new):
    """Rows behind a query's position and blocks that are not listed hold NaN and infinities."""
    heads, group, dim, page, dtype = 2, 4, 64, 32, BF
    c, p = pair(9, heads, dim, page, dtype, kind)
    table, n = i32([[4, 2, 7, 1]]), 3 * page + 5
    hidden = [(1, s) for s in range(5, page)] + [(0, s) for s in range(page)] + [(2, s) for s in range(page)]  # block 1 is not listed
    for i, (at, s) in enumerate(hidden):
        x = [torch.nan, torch.inf, -torch.inf][i % 3]
        if kind == "same":
            c.k[at, :, s], c.v[at, :, s] = x, x
        else:
            c.k_scale[at, :, s], c.v_scale[at, :, s] = x, x
    q, cu = queries(new, heads, group, dim, dtype, 2), i32([0, new])
    check(c, p, q, table, [n], cu, i32([[[0, 2, 3, -1]] * heads] * new))


@pytest.mark.parametrize("kind", ["same", "int8"])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(kind):
    heads, group, dim, page, dtype = 1, 2, 64, 16, FP
    c, p = pair(4, heads, dim, page, dtype, kind)
    table, cu = i32([[2, 0]]), i32([0, 8])
    q = queries(8, heads, group, dim, dtype, 2)
    # row 28 of 32 has a value (or, in 8 bits, a row) that is NaN: of the last eight rows, 24 to 27 do not see it
    if kind == "same":
        c.v[0, 0, 12, 5] = torch.nan
    else:
        c.v_scale[0, 0, 12] = torch.nan
    out, lse = c.attend(q.cuda(), table.cuda(), i32([32]).cuda(), cu=cu.cuda(), return_lse=True)
    bad = out.isnan().any(1).cpu()
    assert not bad[:4].any() and not lse.isnan().any()
    assert bad[4:, 5].all() and (kind == "int8" or not bad[4:, :5].any() and not bad[4:, 6:].any())


def test_scores_at_the_ends():
    """Scores far apart, all the same, and too large for a sum of powers without a maximum."""
    heads, group, dim, page, dtype = 1, 4, 128, 16, BF
    c, p = pair(6, heads, dim, page, dtype, "same")
    q = queries(1, heads, group, dim, dtype, 1)
    table, lens = i32([[0, 1, 2, 3, 4, 5]]), [6 * page - 1]
    for scale in (0.0, -1.0, 30.0, 1e-30):
        check(c, p, q, table, lens, None, None, scale=scale)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scales_far_apart(kind, dtype):
    """Rows in 8 bits whose scales differ by many powers of two, zeros among them, in any order; queries large and small."""
    heads, group, dim, page = 1, 6, 96, 16
    c, p = pair(8, heads, dim, page, dtype, kind)
    g = torch.Generator().manual_seed(3)
    for order in (1, -1):
        scale = torch.exp2(torch.linspace(-14, 6, 8 * page) * order).view(8, 1, page) * torch.rand((8, 1, page), generator=g)
        scale[3, 0, 4:9] = 0
        c.v_scale.copy_(scale)
        p.v_scale.copy_(c.v_scale.cpu().double())
        q = queries(1, heads, group, dim, dtype, 1)
        q[0, 1] *= 64
        q[0, 2] /= 4096
        q[0, 3] = 0
        check(c, p, q, i32([[0, 1, 2, 3, 4, 5, 6, 7]]), [8 * page], None, None)


@pytest.mark.parametrize("kind", ["same", "int8"])
def test_offsets_beyond_32_bits(kind):
    """The last pages of a cache of more than 2^31 values."""
    import ferrolm_b200 as fv

    heads, group, dim, page, dtype = 8, 2, 128, 128, BF
    pages = (1 << 31) // (heads * dim * page) + 40
    c = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind=kind)
    small, p = pair(40, heads, dim, page, dtype, kind, seed=3)
    for name in ("k", "v") + (("k_scale", "v_scale") if kind != "same" else ()):
        getattr(c, name)[-40:].copy_(getattr(small, name))
    table, lens = batch(3, 6, 40, 1), [700, 768, 129]
    q = queries(3, heads, group, dim, dtype, 2)
    far = table + (pages - 40)
    want = p.attend(q, table, lens, None, None, dim**-0.5, q.double(), q[..., 0].double())
    got = c.attend(q.cuda(), far.cuda(), i32(lens).cuda())
    assert ((got.cpu().double() - want[0]).abs() <= want[2]).all()
    # and rows written and read back there
    k, v = rows(3, heads, dim, dtype, 7).cuda(), rows(3, heads, dim, dtype, 8).cuda()
    c.add(k, v, far.cuda(), i32(lens).cuda())
    small.add(k, v, table.cuda(), i32(lens).cuda())
    for name in ("k", "v", "bounds", "bound_codes", "bound_scale"):
        assert torch.equal(getattr(c, name)[-40:].float(), getattr(small, name).float()) or name in ("k", "v")
    assert all(torch.equal(x, y) for x, y in zip(c.vectors(far.cuda(), i32(lens).cuda()), small.vectors(table.cuda(), i32(lens).cuda())))


def test_the_same_result_every_time_and_in_a_graph():
    """Nothing depends on an order that differs between runs; a captured call reads what its tensors hold when it is replayed."""
    heads, group, dim, page, dtype = 2, 4, 128, 64, BF
    c, p = pair(60, heads, dim, page, dtype, "int8")
    table, lens = batch(2, 25, 60, 1).cuda(), i32([1500, 1600]).cuda()
    q = queries(2, heads, group, dim, dtype, 1).cuda()
    first = c.attend(q, table, lens, return_lse=True)
    for _ in range(20):
        assert all(torch.equal(x, y) for x, y in zip(c.attend(q, table, lens, return_lse=True), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blocks = c.search_blocks(q, table, lens, 8)
        out = c.attend(q, table, lens, blocks=blocks)
    for seed in (5, 6):
        q.copy_(queries(2, heads, group, dim, dtype, seed))
        lens.copy_(i32([700 + seed, 1234]))
        graph.replay()
        assert torch.equal(blocks, c.search_blocks(q, table, lens, 8))
        assert torch.equal(out, c.attend(q, table, lens, blocks=blocks))
