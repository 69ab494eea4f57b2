"""KvCache.add and KvCache.vectors against the cache of tests/kv_plain.py.  Everything is compared exactly: codes, scales,
bounds and their codes are the rounded true values (see kv_plain.coded), and what no call may touch keeps its bits."""
import pytest
import torch

from tests.kv_plain import PlainCache

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAMES = ("k", "v", "bounds", "bound_codes", "bound_scale")


def pair(pages, heads, dim, page, dtype, kind, seed=0):
    """The library's cache and the plain one with the same content: random codes everywhere."""
    import ferrolm_b200 as fv

    g = torch.Generator().manual_seed(seed)
    c, p = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind=kind), PlainCache(pages, heads, dim, page, dtype, kind)
    for name in NAMES + (("k_scale", "v_scale") if kind != "same" else ()):
        t = getattr(c, name)
        x = torch.randint(-9, 10, t.shape, generator=g).double()
        if name == "bounds":
            x = x.sort(2).values
        getattr(p, name).copy_(x)
        t.copy_(x.to(t.dtype) if t.dtype != torch.float8_e4m3fn else x.float().to(t.dtype))
    return c, p


def same_state(c, p):
    for name in NAMES + (("k_scale", "v_scale") if c.kind != "same" else ()):
        x, y = getattr(c, name).cpu().double(), getattr(p, name)
        y = y.to(getattr(c, name).dtype).double() if name.endswith("scale") else y
        assert torch.equal(x.nan_to_num(nan=-12345.0), y.nan_to_num(nan=-12345.0)), name


def batch(B, width, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[: B * width].view(B, width).to(torch.int32)


def i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def cuda(x):
    return None if x is None else x.cuda()


def rows(n, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, heads, dim), generator=g) * torch.exp(2 * torch.randn((n, heads, 1), generator=g))
    x[:, :, ::7] *= 8  # channels that stand out, and halves and equal values, where codes have ties
    x[::3] = (x[::3] * 4).round() / 4
    return x.to(dtype)


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,dim,page", [(BF, 5, 128, 16), (FP, 3, 96, 32), (BF, 2, 64, 64), (FP, 1, 128, 128)])
def test_prompts_then_tokens(kind, dtype, heads, dim, page):
    B, width = 4, 6
    c, p = pair(B * width + 5, heads, dim, page, dtype, kind)
    table = batch(B, width, c.pages, 1)
    # prompts of unequal lengths, one of them empty, one ending on a block's border
    new, lens = [1, 0, 3 * page, 2 * page + 5], [1, 3, 3 * page, 2 * page + 5]
    steps = [(new, lens)]
    for i in range(3):  # then pieces that begin inside blocks, one of a single row, one that crosses several blocks
        new = [[page + 3, 2, 0, 1], [1, 1, 1, 1], [0, 2 * page, 7, page - 5]][i]
        lens = [n + m for n, m in zip(lens, new)]
        steps.append((new, lens))
    for s, (new, lens) in enumerate(steps):
        cu = i32([sum(new[:i]) for i in range(B + 1)])
        n = int(cu[-1])
        k, v = rows(n, heads, dim, dtype, 10 + s), rows(n, heads, dim, dtype, 20 + s)
        c.add(k.cuda(), v.cuda(), table.cuda(), i32(lens).cuda(), cu=cu.cuda())
        p.add(k, v, table, lens, cu)
        same_state(c, p)
    # a single row for every sequence, without cu
    lens = [n + 1 for n in lens]
    k, v = rows(B, heads, dim, dtype, 30), rows(B, heads, dim, dtype, 31)
    c.add(k.cuda(), v.cuda(), table.cuda(), i32(lens).cuda())
    p.add(k, v, table, lens)
    same_state(c, p)
    # all rows of all sequences, and the last few of each
    for take in (lens, [min(n, 5) for n in lens], [0, 1, 0, 2]):
        cu = i32([sum(take[:i]) for i in range(B + 1)])
        n = int(cu[-1])
        got = c.vectors(table.cuda(), i32(lens).cuda(), cu=cu.cuda(), rows=n)
        want = p.vectors(table, lens, cu, *torch.zeros((2, n, heads, dim), dtype=torch.float64))
        for x, y in zip(got, want):
            assert torch.equal(x.cpu().double(), y)
    got = c.vectors(table.cuda(), i32(lens).cuda())
    want = p.vectors(table, lens, None, *torch.zeros((2, B, heads, dim), dtype=torch.float64))
    assert torch.equal(got[1].cpu().double(), want[1]) and torch.equal(got[0].cpu().double(), want[0])


@pytest.mark.parametrize("kind", ["same", "int8", "e4m3"])
def test_rows_that_have_no_place_are_skipped(kind):
    """Entries that name no page, positions before the first and behind the table, rows behind the last sequence."""
    heads, dim, page, dtype = 2, 64, 16, BF
    c, p = pair(12, heads, dim, page, dtype, kind)
    table = i32([[3, -1, 5, 7], [1, 2, 12, 2**31 - 1], [-(2**31), 0, 4, 6], [8, 9, 10, 11]])
    new, lens = [60, 40, 20, 90], [60, 70, 15, 90]  # sequence 2 brings five rows more than it has, 3 more than 4 blocks
    cu = i32([0, 60, 100, 120, 210])
    k, v = rows(230, heads, dim, dtype, 1), rows(230, heads, dim, dtype, 2)  # 20 rows behind the last
    c.add(k.cuda(), v.cuda(), table.cuda(), i32(lens).cuda(), cu=cu.cuda())
    p.add(k, v, table, lens, cu)
    same_state(c, p)
    out = torch.full((2, 230, heads, dim), 7.5, dtype=dtype)
    got = c.vectors(table.cuda(), i32(lens).cuda(), cu=cu.cuda(), rows=230, out=tuple(out.cuda().unbind(0)))
    want = p.vectors(table, lens, cu, *out.double().unbind(0))
    for x, y in zip(got, want):
        assert torch.equal(x.cpu().double(), y)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_values_at_the_ends_of_the_type(kind, dtype):
    """Zeros, the smallest and the largest numbers, one value alone, and rows with values that are not finite."""
    heads, dim, page = 1, 64, 16
    c, p = pair(2, heads, dim, page, dtype, kind)
    k = rows(16, heads, dim, dtype, 1)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    k[0] = 0
    k[1] = torch.linspace(-big, big, dim).to(dtype)
    k[2] = small * torch.arange(dim)
    k[3] = 0
    k[3, 0, 5] = -small
    k[4, 0, 3] = torch.inf
    k[5, 0, 3] = torch.nan
    k[6, 0, 3] = -torch.inf
    k[7] = -3.0
    k[8] = small
    k[8, 0, 9] = big
    v = k.flip(0).contiguous()
    table = i32([[1]])
    c.add(k.cuda(), v.cuda(), table.cuda(), i32([16]).cuda(), cu=i32([0, 16]).cuda())
    p.add(k, v, table, [16], i32([0, 16]))
    same_state(c, p)
    got = c.vectors(table.cuda(), i32([16]).cuda(), cu=i32([0, 16]).cuda(), rows=16)
    want = p.vectors(table, [16], i32([0, 16]), *torch.zeros((2, 16, heads, dim), dtype=torch.float64))
    for x, y in zip(got, want):
        assert torch.equal(x.cpu().double().nan_to_num(nan=-5.0), y.nan_to_num(nan=-5.0))


def test_parts_of_a_projection_and_another_stream():
    """Rows with strides of their own, unaligned ones, and a call on a stream that is not the default one."""
    heads, dim, page, dtype = 2, 96, 32, FP
    c, p = pair(4, heads, dim, page, dtype, "int8")
    g = torch.Generator().manual_seed(3)
    both = torch.randn((40, 3 + 2 * heads, dim), generator=g).to(dtype)
    _, k, v = both.split([3, heads, heads], 1)
    odd = torch.randn((40, heads, dim + 1), generator=g).to(dtype)
    table, lens, cu = i32([[2, 0]]), [40], i32([0, 40])
    dk, dv = both.cuda().split([3, heads, heads], 1)[1:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.add(dk, dv, table.cuda(), i32(lens).cuda(), cu=cu.cuda())
        c.add(odd.cuda()[:, :, 1:], dv, table.cuda(), i32(lens).cuda(), cu=cu.cuda())
    s.synchronize()
    p.add(k, v, table, lens, cu)
    p.add(odd[:, :, 1:], v, table, lens, cu)
    same_state(c, p)
    # a head that is the same for all rows and a row that is the same for all heads: strides of zero
    one = torch.randn((40, 1, dim), generator=g).to(dtype)
    c.add(one.cuda().expand(40, heads, dim), dv, table.cuda(), i32(lens).cuda(), cu=cu.cuda())
    p.add(one.expand(40, heads, dim), v, table, lens, cu)
    same_state(c, p)


@pytest.mark.parametrize("B", [31, 33, 70, 1100])
def test_many_sequences(B):
    """Sequences are found among more than fit one look."""
    heads, dim, page, dtype = 1, 64, 16, BF
    c, p = pair(2 * B + 1, heads, dim, page, dtype, "same")
    g = torch.Generator().manual_seed(B)
    table = batch(B, 2, c.pages, B)
    new = torch.randint(0, 20, (B,), generator=g).tolist()
    lens = [n + int(torch.randint(0, 12, (1,), generator=g)) for n in new]
    cu = i32([0] + torch.tensor(new).cumsum(0).tolist())
    n = int(cu[-1])
    k, v = rows(n, heads, dim, dtype, 1), rows(n, heads, dim, dtype, 2)
    c.add(k.cuda(), v.cuda(), table.cuda(), i32(lens).cuda(), cu=cu.cuda())
    p.add(k, v, table, lens, cu)
    same_state(c, p)
    got = c.vectors(table.cuda(), i32(lens).cuda(), cu=cu.cuda(), rows=n)
    assert torch.equal(got[0].cpu(), k) and torch.equal(got[1].cpu(), v)


def test_nothing_to_do():
    import ferrolm_b200 as fv

    c = fv.KvCache(3, 2, 64, page_size=16)
    none = torch.empty((0, 2, 64), dtype=BF, device="cuda")
    table, lens = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    c.add(none, none, table, lens, cu=torch.zeros(3, dtype=torch.int32, device="cuda"))
    c.add(none, none, table[:0], lens[:0])
    assert c.vectors(table, lens, cu=torch.zeros(3, dtype=torch.int32, device="cuda"))[0].shape == (0, 2, 64)
    empty = fv.KvCache(0, 2, 64, page_size=16)
    one = torch.ones((2, 2, 64), dtype=BF, device="cuda")
    empty.add(one, one, table, lens)
    torch.cuda.synchronize()
    assert not c.k.any() and not c.bounds.any()
