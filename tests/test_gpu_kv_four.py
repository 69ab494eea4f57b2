"""The 4-bit cache (kind "int4x32"): rows written and read back exactly, blocks found, attention of tokens and prompts against 64 bits."""
import pytest
import torch

from tests.kv_plain_four import PlainFour, SCALES, coded4, packed4
from tests.test_gpu_kv_attend import check, lists, queries
from tests.test_gpu_kv_rows import batch, cuda, i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
KIND = "int4x32"


def caches(pages, heads, dim, page, dtype):
    import ferrolm_b200 as fv

    return fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind=KIND), PlainFour(pages, heads, dim, page, dtype)


def pair(pages, heads, dim, page, dtype, seed=0):
    """Caches that hold random codes, with scales of several sizes."""
    c, p = caches(pages, heads, dim, page, dtype)
    g = torch.Generator().manual_seed(seed)
    for name in ("k", "v"):
        codes = torch.randint(-7, 8, (pages, heads, page, dim // 32, 32), generator=g).double()
        n = torch.randint(110, 132, codes.shape[:-1], generator=g)  # 2^-5 to 3
        getattr(c, name).copy_(packed4(codes))
        getattr(c, name + "_scale").copy_(n.to(torch.uint8))
        p.hold(name, codes, n)
    return c, p


def special_rows(n, heads, dim, dtype, seed):
    """Rows of every size, with groups of zeros, of the smallest and largest numbers, of ties, and with values that are no numbers."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, heads, dim // 32, 32), generator=g) * torch.exp2(torch.randint(-20, 15, (n, heads, dim // 32, 1), generator=g).float())
    tie = torch.randint(-13, 14, (n, heads, dim // 32, 32), generator=g) / 2.0  # of a scale of 1: 7 is among them
    tie[..., 0] = 7.0
    which = torch.randint(0, 12, (n, heads, dim // 32, 1), generator=g)
    x = torch.where(which == 0, tie * torch.exp2(torch.randint(-17, 13, which.shape, generator=g).float()), x)
    x = torch.where(which == 1, torch.zeros(()), x)
    x = torch.where(which == 2, torch.finfo(dtype).smallest_normal * torch.randint(-3, 4, x.shape, generator=g), x)
    x = torch.where(which == 3, torch.finfo(dtype).max * torch.rand(x.shape, generator=g).round(), x)
    x = x.to(dtype)
    odd = torch.tensor([torch.nan, torch.inf, -torch.inf]).to(dtype)[torch.randint(0, 3, x.shape, generator=g)]
    return torch.where((which == 4) & (torch.rand(x.shape, generator=g) < 0.1), odd, x).flatten(2)


@pytest.mark.parametrize("dtype,heads,dim,page", [(BF, 2, 128, 16), (FP, 3, 96, 32), (BF, 5, 64, 128), (FP, 1, 128, 64), (BF, 3, 96, 16), (FP, 9, 64, 16)])
@pytest.mark.parametrize("news", [[1] * 7, [37, 0, 1, 90, 5], [3, 4, 2, 1]])
def test_rows(dtype, heads, dim, page, news):
    """Written twice, in two pieces, into pages of no order; read back with rows behind the last sequence left as they are."""
    B, width = len(news), 12
    c, p = caches(B * width + 3, heads, dim, page, dtype)
    table, lens = batch(B, width, B * width + 3, 1), [0] * B
    table[-1, 0] = -1
    for step in range(2):
        lens = [a + b for a, b in zip(lens, news)]
        cu = None if set(news) == {1} else i32([0] + torch.tensor(news).cumsum(0).tolist())
        n = sum(news) + (0 if cu is None else 3)
        k, v = special_rows(n, heads, dim, dtype, 5 + step), special_rows(n, heads, dim, dtype, 9 + step)
        c.add(k.cuda(), v.cuda(), table.cuda(), i32(lens).cuda(), cu=cuda(cu))
        p.add(k, v, table, lens, cu)
        got = c.vectors(table.cuda(), i32(lens).cuda(), cu=cuda(cu), rows=n, out=tuple(torch.full((n, heads, dim), 3.25, dtype=dtype, device="cuda") for _ in range(2)))
        want = p.vectors(table, lens, cu, *(torch.full((n, heads, dim), 3.25, dtype=torch.float64) for _ in range(2)))
        for x, y in zip(got, want):
            assert torch.equal(x.cpu().double().nan_to_num(nan=-9e9), y.nan_to_num(nan=-9e9))
    for name in ("bounds", "bound_codes"):
        assert torch.equal(getattr(c, name).cpu().double(), getattr(p, name)), name
    assert torch.equal(c.bound_scale.cpu(), p.bound_scale.float())


@pytest.mark.parametrize("dim", [64, 96, 128])
def test_where_codes_and_scales_lie(dim):
    """The bytes that the header describes."""
    c, _ = caches(3, 2, dim, 16, BF)
    k, v = special_rows(40, 2, dim, BF, 1), special_rows(40, 2, dim, BF, 2)
    c.add(k.cuda(), v.cuda(), i32([[2, 0, 1]]).cuda(), i32([40]).cuda(), cu=i32([0, 40]).cuda())
    for x, held, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        codes, n = coded4(x.double())
        at, slot = torch.tensor([2, 0, 1])[torch.arange(40) // 16], torch.arange(40) % 16
        assert torch.equal(held.cpu()[at, :, slot], packed4(codes))
        assert torch.equal(scale.cpu()[at, :, slot].long(), n)
    assert float(SCALES[225]) == 9216.0 and len(SCALES) == 226


@pytest.mark.parametrize("dtype", [BF, FP])
def test_values_are_within_half_a_step(dtype):
    """Of a scale that is at most an eighth above a seventh of the largest value."""
    c, _ = caches(20, 4, 128, 64, dtype)
    x = (torch.randn((1000, 4, 128)) * torch.exp(torch.randn((1000, 4, 1)))).to(dtype).cuda()
    table, lens, cu = torch.arange(16, dtype=torch.int32).view(1, 16).cuda(), i32([1000]).cuda(), i32([0, 1000]).cuda()
    c.add(x, -x, table, lens, cu=cu)
    k, v = c.vectors(table, lens, cu=cu, rows=1000)
    most = x.float().unflatten(-1, (4, 32)).abs().amax(-1, keepdim=True)
    assert ((k - x).float().unflatten(-1, (4, 32)).abs() <= most * (1.125 / 14)).all() and torch.equal(k, -v)


def test_blocks_are_those_of_a_16_bit_cache():
    import ferrolm_b200 as fv

    four, _ = caches(80, 2, 128, 32, BF)
    same = fv.KvCache(80, 2, 128, page_size=32, dtype=BF)
    table, lens, cu = batch(2, 40, 80, 1).cuda(), i32([1200, 900]).cuda(), i32([0, 1200, 2100]).cuda()
    k, q = torch.randn((2100, 2, 128)).to(BF).cuda(), torch.randn((2100, 6, 128)).to(BF).cuda()
    for x in (four, same):
        x.add(k, k, table, lens, cu=cu)
    assert torch.equal(four.search_blocks(q, table, lens, 9, cu=cu), same.search_blocks(q, table, lens, 9, cu=cu))


@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 3, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 2, 1, 128, 32), (BF, 1, 37, 96, 16), (FP, 1, 8, 64, 16), (BF, 1, 9, 128, 64)])
def test_tokens(dtype, heads, group, dim, page):
    """A row for every sequence: no rows at all, one, a border's neighbours, and enough for several warps and CTAs."""
    lens = [0, 1, 15, 16, 17, page, page + 1, 9 * page - 3, 30 * page]
    c, p = pair(300, heads, dim, page, dtype)
    table = batch(len(lens), 30, 300, 2)
    table[7, 3] = -1
    q = queries(len(lens), heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, None, None)
    check(c, p, q, table, lens, None, lists(len(lens), heads, 11, 30, 4), scale=0.21)
    check(c, p, q, table, lens, None, lists(len(lens), heads, 5, 30, 4), scale=0.0)


@pytest.mark.parametrize("B,blocks", [(1, 40), (1, 9), (3, 130), (40, 3)])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_few_and_many_rows(B, blocks, dim):
    """Every way to cut the work."""
    heads, group, page, dtype = 2, 5, 32, BF
    c, p = pair(B * blocks + 3, heads, dim, page, dtype, seed=B)
    table = batch(B, blocks, c.pages, 2)
    lens = [blocks * page - 7 * b % (blocks * page) for b in range(B)]
    q = queries(B, heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, None, None)
    check(c, p, q, table, lens, None, lists(B, heads, 70, blocks, 5))


@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 1, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 2, 1, 128, 32), (BF, 1, 37, 96, 16), (FP, 1, 3, 64, 32)])
def test_prompts(dtype, heads, group, dim, page):
    """Ragged pieces of prompts, one from the first row on, one that brings more rows than its sequence has, one of no rows, and
    rows behind the last sequence; all blocks, lists of a few, and lists that have nothing in common."""
    news, lens = [40, 0, 13, 9, 25], [40, 5, 13 * page - 3, 6, 200]
    c, p = pair(120, heads, dim, page, dtype)
    table = batch(5, 20, 120, 2)
    table[4, 1] = 4096
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = int(cu[-1]) + 6
    q = queries(n, heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, cu, None)
    check(c, p, q, table, lens, cu, lists(n, heads, 7, 13, 4), scale=-0.17)
    check(c, p, q, table, lens, cu, lists(n, heads, 3, 13, 5))
    check(c, p, q, table[:, :2], lens, cu, None)  # rows behind the table's last column


@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 1, 4, 128, 16), (FP, 2, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 1, 2, 128, 32)])
@pytest.mark.parametrize("news,lens", [([6], [2500]), ([9, 5, 0, 7], [1900, 3, 700, 1025]), ([40, 6], [600, 1700])])
def test_few_rows_over_long_sequences(dtype, heads, group, dim, page, news, lens):
    """Rows of a sequence whose keys are shared out to many CTAs, some of which see nothing; with a result's place given and without,
    with and without the logarithms, rows of no sequence left as they were; and the same without room for it."""
    import ferrolm_b200 as fv

    width = -(-max(lens) // page) + 3
    c, p = pair(width * len(news) + 1, heads, dim, page, dtype, seed=len(news))
    table = batch(len(news), width, c.pages, 2)
    table[0, 2] = -1
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = int(cu[-1]) + 2
    q = queries(n, heads, group, dim, dtype, 3)
    got = check(c, p, q, table, lens, cu, None)
    check(c, p, q, table, lens, cu, lists(n, heads, 60, width, 4))
    at = q.cuda(), table.cuda(), i32(lens).cuda(), cuda(cu)
    alone = c.attend(*at[:3], cu=at[3])
    assert torch.equal(alone[: int(cu[-1])], got[0][: int(cu[-1])])
    # the entry point without work: one CTA for each tile of queries
    whole, lse = torch.zeros_like(got[0]), torch.zeros_like(got[1])
    b = c._batch(at[1], at[2], at[3], n)
    assert fv.kv.lib().fv_kv_attend_work(c._ref, b, group) > 0
    fv.kv.check(c._attend(c._ref, torch.cuda.current_stream().cuda_stream, b, at[0].data_ptr(), at[0].stride(0), at[0].stride(1), group, None, 0, dim**-0.5, whole.data_ptr(), lse.data_ptr(), None, 0))
    want = p.attend(q, table, lens, cu, None, dim**-0.5, torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64))
    assert ((whole.cpu().double() - want[0]).abs() <= want[2]).all()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("news", [[1, 1, 1], [90, 20, 30]])
def test_groups_that_are_no_numbers(dtype, news):
    """A key's reaches every query that sees it, a value's only the components of its group; neither those that do not see it."""
    heads, group, dim, page = 2, 3, 96, 16
    lens = [100, 60, 81]
    c, p = pair(30, heads, dim, page, dtype)
    table = batch(3, 8, 30, 2)
    for name, b, pos, h, g in (("k", 0, 99, 0, 2), ("v", 0, 40, 1, 0), ("v", 1, 59, 0, 1), ("k", 2, 85, 1, 0), ("v", 2, 88, 0, 2), ("v", 2, 64, 1, 1)):
        page_at = int(table[b, pos // page])
        getattr(c, name + "_scale")[page_at, h, pos % page, g] = 255
        getattr(p, name)[page_at, h, pos % page, 32 * g : 32 * g + 32] = torch.nan
    cu = None if news == [1, 1, 1] else i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = sum(news)
    q = queries(n, heads, group, dim, dtype, 3)
    got = check(c, p, q, table, lens, cu, None)[0]
    assert got.isnan().any() and not got.isnan().all()
    check(c, p, q, table, lens, cu, lists(n, heads, 4, 7, 4))


@pytest.mark.parametrize("new", [1, 30])
def test_scales_at_both_ends(new):
    """The smallest scales next to the largest, and queries that are next to nothing or far out."""
    heads, group, dim, page, dtype = 1, 4, 128, 32, BF
    c, p = pair(12, heads, dim, page, dtype)
    g = torch.Generator().manual_seed(4)
    for name, choice in (("k", [1, 2, 9, 100, 120]), ("v", [0, 1, 3, 7, 8, 15, 120, 216, 225])):
        n = torch.tensor(choice)[torch.randint(0, len(choice), (12, 1, page, 4), generator=g)]
        codes = torch.randint(-7, 8, (12, 1, page, 4, 32), generator=g).double()
        getattr(c, name).copy_(packed4(codes)), getattr(c, name + "_scale").copy_(n.to(torch.uint8)), p.hold(name, codes, n)
    table, lens = batch(2, 6, 12, 2), [190, 150]
    cu = None if new == 1 else i32([0, new, 2 * new])
    for by in (1.0, 2.0**-60, 64.0):
        q = (queries(2 * new, heads, group, dim, torch.float32, 3) * by).to(dtype)
        check(c, p, q, table, lens, cu, None)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_few_rows_and_groups_that_are_no_numbers(dtype):
    """Keys shared out to many CTAs: a key's reaches every query that sees it, whichever CTA has it, a value's its group only."""
    heads, group, dim, page, lens, news = 2, 4, 128, 32, [3000, 2200], [6, 5]
    c, p = pair(190, heads, dim, page, dtype)
    table, cu = batch(2, 94, 190, 2), i32([0, 6, 11])
    for name, b, pos, h, g in (("v", 0, 2996, 0, 2), ("v", 0, 17, 1, 1), ("k", 1, 2197, 0, 0), ("v", 1, 1500, 1, 3)):
        at = int(table[b, pos // page])
        getattr(c, name + "_scale")[at, h, pos % page, g] = 255
        getattr(p, name)[at, h, pos % page, 32 * g : 32 * g + 32] = torch.nan
    q = (queries(11, heads, group, dim, torch.float32, 3) * 0.1).to(dtype)  # weights of all rows
    got = check(c, p, q, table, lens, cu, None)[0]
    assert got[:2, :group, 64:96].isfinite().all() and got[3:6, :group, 64:96].isnan().all() and got[:6, group:, 32:64].isnan().all()
    assert got[6:8, :group].isfinite().all() and got[8:, :group].isnan().all()


def test_few_rows_captured_and_on_two_streams():
    """Each call has its parts' place to itself."""
    heads, group, dim, page = 2, 4, 128, 64
    c, _ = pair(200, heads, dim, page, BF)
    table, cu = batch(2, 90, 200, 2).cuda(), i32([0, 6, 12]).cuda()
    q = [queries(12, heads, group, dim, BF, i).cuda() for i in range(2)]
    lens, outs = i32([5000, 3000]).cuda(), [torch.zeros_like(x) for x in q]
    for x, out in zip(q, outs):
        c.attend(x, table, lens, cu=cu, out=out)
    graphs = [torch.cuda.CUDAGraph() for _ in q]
    for g, x, out in zip(graphs, q, outs):
        with torch.cuda.graph(g):
            c.attend(x, table, lens, cu=cu, out=out)
    streams = [torch.cuda.Stream() for _ in q]
    for n in (4000, 5700, 300):
        lens.copy_(i32([n, n - 200]))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for x, out in zip(q, outs):
            assert torch.equal(out, c.attend(x, table, lens, cu=cu))


def test_attention_is_that_of_the_rows_read_back():
    """4-bit rows are exact in 16 bits: a 16-bit cache of what vectors gives has the same values, and the results are as near as two ways
    of rounding weights, 2^-9 and 2^-11 of each, and the result are."""
    import ferrolm_b200 as fv

    heads, group, dim, page, n = 2, 4, 128, 64, 3000
    four, _ = caches(60, heads, dim, page, BF)
    same = fv.KvCache(60, heads, dim, page_size=page, dtype=BF)
    table, lens, cu = batch(1, 50, 60, 1).cuda(), i32([n]).cuda(), i32([0, n]).cuda()
    rows = torch.randn((n, heads * (group + 2), dim)).to(BF).cuda()
    q, k, v = rows.split([heads * group, heads, heads], 1)
    four.add(k, v, table, lens, cu=cu)
    same.add(*four.vectors(table, lens, cu=cu, rows=n), table, lens, cu=cu)
    for at in (slice(0, n), slice(n - 1, n)):
        c = i32([0, len(range(n)[at])]).cuda()
        x, y = (z.attend(q[at], table, lens, cu=c, return_lse=True) for z in (four, same))
        most = float(v.float().abs().max())
        assert (x[0] - y[0]).abs().max() <= (2.0**-9 + 2.0**-11 + 2 * 2.0**-9) * 1.1 * most
        assert (x[1] - y[1]).abs().max() <= 2.0**-14


def test_a_captured_call():
    heads, group, dim, page = 2, 4, 128, 64
    c, p = pair(70, heads, dim, page, BF)
    table, q = batch(2, 30, 70, 2).cuda(), queries(2, heads, group, dim, BF, 3).cuda()
    lens, out = i32([500, 1800]).cuda(), torch.zeros((2, heads * group, dim), dtype=BF, device="cuda")
    k = torch.randn((2, heads, dim)).to(BF).cuda()

    def step():
        c.add(k, k, table, lens)
        c.attend(q, table, lens, out=out)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for more in (1, 2, 15):
        lens.copy_(i32([500 + more, 1800 + more]))
        k.normal_()
        graph.replay()
        got = out.clone()
        assert torch.equal(got, c.attend(q, table, lens))
