"""KvCache.search_blocks against the cache of tests/kv_plain.py.  Scores are whole numbers times a scale, so the blocks are
compared exactly, whichever way the work was cut."""
import pytest
import torch

from tests.kv_plain import PlainCache
from tests.test_gpu_kv_rows import batch, cuda, i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def pair(pages, heads, dim, page, dtype, seed=0, ties=False):
    """Caches with random bounds; `ties`: of a few values only, so that many blocks have the same score."""
    import ferrolm_b200 as fv

    g = torch.Generator().manual_seed(seed)
    c, p = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype), PlainCache(pages, heads, dim, page, dtype, "same")
    if ties:
        some = torch.randint(-127, 128, (3, heads, 2, dim), generator=g).double()
        at = torch.randint(0, 3, (pages,), generator=g)
        p.bound_codes.copy_(some[at])
        p.bound_scale.copy_((at.double() + 1)[:, None].expand(pages, heads))
    else:
        p.bound_codes.copy_(torch.randint(-127, 128, p.bound_codes.shape, generator=g))
        p.bound_scale.copy_(torch.rand(p.bound_scale.shape, generator=g))
    c.bound_codes.copy_(p.bound_codes.to(torch.int8))
    c.bound_scale.copy_(p.bound_scale.float())
    p.bound_scale.copy_(p.bound_scale.float())
    return c, p


def queries(n, heads, group, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((n, heads * group, dim), generator=g).to(dtype)


def check(c, p, q, table, lens, k, cu, first=1, recent=2, rows=None):
    n = q.shape[0] if rows is None else rows
    out = torch.full((q.shape[0], c.heads, k), -7, dtype=torch.int64)
    want = p.search(q, table, lens, k, cu, first, recent, out.clone())
    got = c.search_blocks(q.cuda(), table.cuda(), i32(lens).cuda(), k, cu=cuda(cu), first=first, recent=recent, out=out.int().cuda())
    assert torch.equal(got.cpu().long(), want), (k, first, recent)
    return n


@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 3, 7, 96, 64), (BF, 1, 16, 64, 128), (FP, 2, 1, 128, 32), (BF, 1, 37, 64, 16)])
@pytest.mark.parametrize("ties", [False, True])
def test_tokens(dtype, heads, group, dim, page, ties):
    """A row for every sequence: no block at all, one, some, and a whole table of them."""
    lens = [0, 1, page, page + 1, 9 * page - 3, 40 * page, 70 * page]
    c, p = pair(500, heads, dim, page, dtype, ties=ties)
    table = batch(len(lens), 70, 500, 2)
    q = queries(len(lens), heads, group, dim, dtype, 3)
    for k, first, recent in ((1, 0, 0), (1, 1, 2), (4, 1, 2), (9, 0, 1), (33, 3, 5), (100, 1, 2)):
        check(c, p, q, table, lens, k, None, first, recent)


@pytest.mark.parametrize("heads,group,dim,page,new", [(2, 4, 128, 16, 45), (1, 3, 96, 32, 100), (1, 8, 64, 16, 7)])
@pytest.mark.parametrize("ties", [False, True])
def test_prompts(heads, group, dim, page, new, ties):
    """Rows of ragged pieces of prompts, some without any, with rows behind the last sequence."""
    news, lens = [new, 0, 1, new + 13, 5], [new, 4, 30 * page, 900, 2]  # the last one has fewer rows than it brings
    c, p = pair(400, heads, dim, page, BF, ties=ties)
    table = batch(5, 60, 400, 2)
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    q = queries(int(cu[-1]) + 11, heads, group, dim, BF, 3)
    for k, first, recent in ((6, 1, 2), (20, 0, 0)):
        check(c, p, q, table, lens, k, cu, first, recent)


@pytest.mark.parametrize("width", [130, 500, 700, 1500, 3200, 7000])
@pytest.mark.parametrize("new", [1, 21])
def test_long_sequences(width, new):
    """Every width at which another number of rows shares a CTA, and keys that stay in registers or do not."""
    heads, group, dim, page = 1, 2, 64, 16
    c, p = pair(width + 9, heads, dim, page, BF, seed=width)
    table = batch(1, width, width + 9, 2)
    q = queries(new, heads, group, dim, BF, 3)
    check(c, p, q, table, [width * page - 5], 24, i32([0, new]))
    check(c, p, q, table, [width * page - 5], width // 2, i32([0, new]), 5, 7)


def test_blocks_without_a_page_and_behind_the_table():
    heads, group, dim, page = 2, 2, 64, 16
    c, p = pair(9, heads, dim, page, FP)
    table = i32([[0, -1, 2, 9, 4, 2**31 - 1, 6, -(2**31)], [8, 7, 6, 5, 4, 3, 2, 1], [-1] * 8])
    q = queries(3, heads, group, dim, FP, 1)
    for lens in ([8 * page, 8 * page + 100, 8 * page], [5 * page, 1, 0]):
        for k in (2, 3, 8):
            check(c, p, q, table, lens, k, None)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_queries_at_the_ends_of_the_type(dtype):
    """Zeros (every score the same), the largest and smallest values, infinities and NaN, which count as zero."""
    heads, group, dim, page = 1, 2, 64, 16
    c, p = pair(30, heads, dim, page, dtype)
    c.bound_scale[3:6], p.bound_scale[3:6] = 0.0, 0.0  # blocks of zeros: scores of +0 and -0 are equal
    q = queries(7, heads, group, dim, dtype, 1)
    q[0] = 0
    q[1] = torch.finfo(dtype).max * torch.linspace(-1, 1, 2 * dim).view(2, dim).to(dtype)
    q[2] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * (torch.arange(2 * dim).view(2, dim) - 60)
    q[3, 0, 5], q[4, 1, 6], q[5, 0, 7] = torch.nan, torch.inf, -torch.inf
    q[6] = torch.nan
    for k in (4, 11):
        check(c, p, q, batch(7, 4, 30, 1), [4 * page] * 7, k, None, 0, 0)
        check(c, p, q, batch(1, 30, 30, 1), [30 * page], k, i32([0, 7]), 0, 1)


def test_the_same_blocks_whichever_way_the_rows_are_cut():
    """A piece of a prompt at once, by rows, and as parts of longer rows on another stream."""
    heads, group, dim, page = 4, 4, 128, 64
    c, _ = pair(300, heads, dim, page, BF, seed=5)
    table, q = batch(1, 260, 300, 1).cuda(), queries(200, heads, group, dim, BF, 2).cuda()
    n = 260 * page - 9
    whole = c.search_blocks(q, table, i32([n]).cuda(), 16, cu=i32([0, 200]).cuda())
    rows = torch.cat([c.search_blocks(q[i : i + 1], table, i32([n - 199 + i]).cuda(), 16) for i in range(200)])
    assert torch.equal(whole, rows)
    wide = torch.zeros((200, heads * group + 5, dim), dtype=BF, device="cuda")
    wide[:, 5:] = q
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = c.search_blocks(wide[:, 5:], table, i32([n]).cuda(), 16, cu=i32([0, 200]).cuda())
    s.synchronize()
    assert torch.equal(again, whole)


def test_the_longest_table():
    """As many blocks as one search takes, for a cluster's one row and for rows of a prompt, most of them without a page."""
    heads, group, dim, page, width = 1, 1, 64, 16, 50_000
    c, p = pair(700, heads, dim, page, BF, seed=9)
    table = torch.full((1, width), -1, dtype=torch.int32)
    at = torch.randperm(width, generator=torch.Generator().manual_seed(2))[:690]
    table[0, at] = torch.randperm(700, generator=torch.Generator().manual_seed(3))[:690].to(torch.int32)
    table[0, width - 1], table[0, 0] = 0, 1
    n = width * page - 2
    q = queries(6, heads, group, dim, BF, 3)
    whole = c.search_blocks(q.cuda(), table.cuda(), i32([n]).cuda(), 40, cu=i32([0, 6]).cuda())
    want = p.search(q[5:], table, [n], 40, None, 1, 2, torch.zeros((1, heads, 40), dtype=torch.int64))
    assert torch.equal(whole[5:].cpu().long(), want)
    for i in range(6):
        assert torch.equal(c.search_blocks(q[i : i + 1].cuda(), table.cuda(), i32([n - 5 + i]).cuda(), 40), whole[i : i + 1])


def test_calls_that_are_refused():
    import ferrolm_b200 as fv

    c = fv.KvCache(8, 2, 64, page_size=16)
    table, lens = i32([[0, 1, 2]]).cuda(), i32([40]).cuda()
    q = torch.zeros((1, 4, 64), dtype=BF, device="cuda")
    for bad in (dict(k=0), dict(k=4097), dict(first=-1), dict(recent=-2), dict(lens=lens.long()), dict(table=table[0]), dict(lens=i32([40, 1]).cuda()),
                dict(cu=i32([0, 1, 2]).cuda()), dict(cu=i32([0, 1])), dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.cpu()),
                dict(q=q.expand(2, 4, 64)), dict(q=q.clone().requires_grad_()), dict(out=torch.zeros((1, 2, 5), dtype=torch.int32, device="cuda"))):
        a = dict(q=q, table=table, lens=lens, k=2) | bad
        with pytest.raises(fv.FerrovecError):
            c.search_blocks(a.pop("q"), a.pop("table"), a.pop("lens"), a.pop("k"), **a)
    k = torch.zeros((1, 2, 64), dtype=BF, device="cuda")
    for bad in (dict(k=k.half()), dict(v=k[:, :1]), dict(k=k.expand(2, 2, 64)), dict(table=table.cpu()), dict(v=k.clone().requires_grad_())):
        a = dict(k=k, v=k, table=table, lens=lens) | bad
        with pytest.raises(fv.FerrovecError):
            c.add(**a)
    for bad in (dict(blocks=i32([[[0], [1]]])), dict(blocks=i32([[[0, 1]]]).cuda()), dict(blocks=torch.zeros((1, 2, 0), dtype=torch.int32, device="cuda")),
                dict(scale=float("nan")), dict(out=q.half()), dict(out=(q, q), return_lse=True)):
        with pytest.raises(fv.FerrovecError):
            c.attend(q, table, lens, **bad)
    with pytest.raises(fv.FerrovecError):
        c.vectors(table, lens, out=(k, k.half()))
    with torch.no_grad():  # where no gradient is wanted, a parameter is a tensor like another
        c.attend(q.clone().requires_grad_(), table, lens)
