"""KvCache at the ends of what its calls take: as many forced blocks as a table has, lengths at the ends of 32 bits, the widest table."""
import pytest
import torch

from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def guarded(shape, value, guard, dtype=torch.int32):
    """A tensor between two stretches of `guard` numbers: (the whole, the tensor)."""
    n = torch.Size(shape).numel()
    whole = torch.full((guard + n + guard,), value, dtype=dtype, device="cuda")
    return whole, whole[guard : guard + n].view(shape)


@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("first,recent", [(32_767, 0), (32_768, 0), (50_000, 0), (0, 32_767), (0, 32_768), (0, 40_000), (0, 50_000), (16_384, 16_384), (25_000, 25_000), (2**40, 2**40)])
def test_more_forced_blocks_than_half_a_word_counts(first, recent, new):
    """The longest table, all of its blocks there, and more of them forced than the result has room for: the lowest of the forced ones
    are the result, and nothing is written before or behind it."""
    import ferrolm_b200 as fv

    heads, dim, page, width = 2, 64, 16, 50_000
    g = torch.Generator().manual_seed(first + recent)
    c = fv.KvCache(700, heads, dim, page_size=page)
    c.bound_codes.copy_(torch.randint(-127, 128, c.bound_codes.shape, generator=g))
    c.bound_scale.copy_(torch.rand(c.bound_scale.shape, generator=g))
    table = torch.randint(0, 700, (1, width), generator=g).to(torch.int32).cuda()
    q = torch.randn((new, heads, dim), generator=g).to(BF).cuda()
    length = width * page - 2
    last = torch.tensor([(length - new + i) // page for i in range(new)])
    for k in (1, 32, 128, 129, 256, 300, 4096):
        whole, out = guarded((new, heads, k), -7, 60_000)
        c.search_blocks(q, table, i32([length]).cuda(), k, cu=i32([0, new]).cuda(), first=first, recent=recent, out=out)
        begin = torch.zeros_like(last) if first else (last - recent + 1).clamp(min=0)
        want = begin[:, None] + torch.arange(k)[None]
        assert torch.equal(out.cpu().long(), want[:, None].expand(new, heads, k)), k
        assert (whole[:60_000] == -7).all() and (whole[60_000 + out.numel() :] == -7).all(), k


@pytest.mark.parametrize("kind", ["same", "int8"])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("blocks", [6, 300])
def test_lengths_below_zero_are_sequences_without_rows(kind, new, blocks):
    """As low as 32 bits go, where a position before the first would come out as one behind the last; beside a sequence that has rows."""
    import ferrolm_b200 as fv

    heads, group, dim, page = 2, 2, 64, 16
    g = torch.Generator().manual_seed(new)
    c = fv.KvCache(2 * blocks, heads, dim, page_size=page, kind=kind)
    pages = torch.randperm(2 * blocks, generator=g).view(2, blocks).to(torch.int32).cuda()
    live = 5 * page + 3
    first = torch.randn((live, heads, dim), generator=g).to(BF).cuda()
    c.add(first, first, pages[1:], i32([live]).cuda(), cu=i32([0, live]).cuda())
    rows = torch.randn((2 * new, heads * (group + 2), dim), generator=g).to(BF).cuda()
    q, k, v = rows.split([heads * group, heads, heads], 1)
    names = ("k", "v", "bounds", "bound_codes", "bound_scale") + (("k_scale", "v_scale") if kind != "same" else ())
    cu = i32([0, new, 2 * new]).cuda() if new > 1 else None
    alone = i32([0, new]).cuda() if new > 1 else None
    before = {n: getattr(c, n).clone() for n in names}
    c.add(k[new:], v[new:], pages[1:], i32([live]).cuda(), cu=alone)
    after = {n: getattr(c, n).clone() for n in names}
    want = [c.search_blocks(q[new:], pages[1:], i32([live]).cuda(), 4, cu=alone), *c.attend(q[new:], pages[1:], i32([live]).cuda(), cu=alone, return_lse=True)]
    for low in (-(2**31), -(2**31) + 1, -(2**31) + new, -1, 0):
        lens = i32([low, live]).cuda()
        for n in names:
            getattr(c, n).copy_(before[n])
        c.add(k, v, pages, lens, cu=cu)
        for n in names:
            assert torch.equal(getattr(c, n).float(), after[n].float()), (n, low)
        out = torch.full((2, 2 * new, heads, dim), 7.5, dtype=BF, device="cuda")
        c.vectors(pages, lens, cu=cu, rows=2 * new, out=tuple(out.unbind(0)))
        assert (out[:, :new] == 7.5).all() and (out[:, new:] != 7.5).any()
        blocks_found = c.search_blocks(q, pages, lens, 4, cu=cu)
        assert (blocks_found[:new] == -1).all() and torch.equal(blocks_found[new:], want[0])
        for lists in (None, torch.arange(4, dtype=torch.int32, device="cuda").expand(2 * new, heads, 4).contiguous()):
            got, lse = c.attend(q, pages, lens, cu=cu, blocks=lists, return_lse=True)
            assert (got[:new] == 0).all() and (lse[:new] == -torch.inf).all(), low
            if lists is None:  # the work may be cut in other places: weights and results are rounded twice on both sides, half a step of bf16 each
                assert (got[new:].float() - want[1].float()).abs().max() <= 4 * 2.0**-8 * want[1].float().abs().max()
                assert (lse[new:] - want[2]).abs().max() <= 2.0**-12


@pytest.mark.parametrize("kind", ["same", "e4m3"])
def test_the_tensors_of_a_cache_stay(kind):
    """Another tensor in place of one that every call's address is from would leave the calls with memory that is freed."""
    import ferrolm_b200 as fv

    c = fv.KvCache(3, 2, 64, page_size=16, kind=kind)
    for name in ("k", "v", "bounds", "bound_codes", "bound_scale", "k_scale", "v_scale"):
        x = getattr(c, name)
        assert (x is None) == (kind == "same" and name.endswith("_scale") and name != "bound_scale")
        with pytest.raises(AttributeError):
            setattr(c, name, None if x is None else x.clone())
        assert getattr(c, name) is x
    pool = {n: getattr(c, n) for n in ("k", "v", "bounds", "bound_codes", "bound_scale", "k_scale", "v_scale")}
    again = fv.KvCache(3, 2, 64, page_size=16, kind=kind, buffers=pool)
    assert all(getattr(again, n) is x for n, x in pool.items())


@pytest.mark.parametrize("kind,dtype", [("same", BF), ("same", torch.float16), ("int8", BF), ("e4m3", torch.float16)])
@pytest.mark.parametrize("group", [100, 128])
def test_the_largest_groups(kind, dtype, group):
    """One row to a tile of a prompt, several tiles of queries to a row by itself, and the largest sums of a search."""
    from tests.test_gpu_kv_attend import check, lists, pair, queries
    from tests.test_gpu_kv_search import check as check_search

    heads, dim, page = 2, 64, 16
    c, p = pair(30, heads, dim, page, dtype, kind)
    table = torch.randperm(30, generator=torch.Generator().manual_seed(1))[:28].view(2, 14).to(torch.int32)
    for news, lens in (([7, 6], [14 * page - 3, 40]), ([1, 1], [100, 9 * page])):
        cu, n = i32([0, news[0], sum(news)]), sum(news)
        q = queries(n, heads, group, dim, dtype, 3)
        check(c, p, q, table, lens, cu, None)
        check(c, p, q, table, lens, cu, lists(n, heads, 5, 9, 4))
    x = torch.randint(-127, 128, p.bound_codes.shape, generator=torch.Generator().manual_seed(2))
    p.bound_codes.copy_(x), c.bound_codes.copy_(x.to(torch.int8))
    p.bound_scale.fill_(0.25), c.bound_scale.fill_(0.25)
    q = torch.full((13, heads * group, dim), 3.0, dtype=dtype)  # all codes 127: sums of 127 * group
    q[5:, ::2] = -3.0
    q[9:, :, ::3] = 0.01
    check_search(c, p, q, table, [14 * page - 3, 9 * page], 4, i32([0, 7, 13]))


@pytest.mark.parametrize("kind", ["same", "int8"])
@pytest.mark.parametrize("new", [1, 9])
def test_nothing_to_look_at(kind, new):
    """No column in the table, no page in the cache, no entry that is a page, no row that belongs to a sequence: zeros, -inf and -1 for rows
    of sequences, and rows of none are left alone."""
    import ferrolm_b200 as fv

    heads, group, dim, page, B = 3, 4, 96, 32, 2
    rows = torch.randn((B * new + 3, heads * (group + 2), dim), device="cuda").to(BF)
    q, k, v = rows.split([heads * group, heads, heads], 1)
    lens, cu, none = i32([500, 700]).cuda(), i32([0, new, 2 * new]).cuda(), i32([0, 0, 0]).cuda()
    full = torch.arange(40, dtype=torch.int32, device="cuda").view(B, 20)
    for pages, table, at in ((40, full[:, :0], cu), (0, full, cu), (40, torch.full_like(full, -1), cu), (40, full, none), (0, full[:, :0], none)):
        c = fv.KvCache(pages, heads, dim, page_size=page, kind=kind)
        c.add(k, v, table, lens, cu=at)
        assert not c.k.any() and not c.bounds.any()
        out = torch.full((2, len(q), heads, dim), 7.5, dtype=BF, device="cuda")
        c.vectors(table, lens, cu=at, out=tuple(out.unbind(0)))
        assert at is none or (out == 7.5).all()
        found = torch.full((len(q), heads, 6), -9, dtype=torch.int32, device="cuda")
        c.search_blocks(q, table, lens, 6, cu=at, out=found)
        live = 0 if at is none else 2 * new
        assert (found[:live] == -1).all() and (found[live:] == -9).all()
        for lists in (None, torch.arange(6, dtype=torch.int32, device="cuda").expand(len(q), heads, 6).contiguous()):
            y, lse = torch.full_like(q, 7.5).contiguous(), torch.full((len(q), heads * group), 7.5, device="cuda")
            c.attend(q, table, lens, cu=at, blocks=lists, return_lse=True, out=(y, lse))
            assert (y[:live] == 0).all() and (lse[:live] == -torch.inf).all() and (y[live:] == 7.5).all() and (lse[live:] == 7.5).all()


@pytest.mark.parametrize("kind,dtype", [("same", BF), ("int8", torch.float16)])
@pytest.mark.parametrize("piece", [50, 70])
def test_single_rows_and_a_piece_of_a_prompt_in_one_call(kind, dtype, piece):
    """20 sequences of a row each around one that brings 50 rows (all of them go by themselves) or 70 (all go as prompts)."""
    from tests.test_gpu_kv_attend import check, lists, pair, queries
    from tests.test_gpu_kv_search import check as check_search

    heads, group, dim, page, B = 2, 4, 64, 16, 21
    c, p = pair(B * 8, heads, dim, page, dtype, kind)
    g = torch.Generator().manual_seed(piece)
    table = torch.randperm(B * 8, generator=g).view(B, 8).to(torch.int32)
    news = [1] * 9 + [piece] + [1] * 11
    lens = [int(torch.randint(1, 8 * page, (1,), generator=g)) for _ in news]
    lens[9], lens[3], lens[15] = 8 * page - 1, 1, 0
    cu = i32([0] + torch.tensor(news).cumsum(0).tolist())
    n = int(cu[-1])
    q = queries(n, heads, group, dim, dtype, 3)
    check(c, p, q, table, lens, cu, None)
    check(c, p, q, table, lens, cu, lists(n, heads, 4, 8, 4))
    x = torch.randint(-127, 128, p.bound_codes.shape, generator=g)
    p.bound_codes.copy_(x), c.bound_codes.copy_(x.to(torch.int8))
    p.bound_scale.fill_(0.25), c.bound_scale.fill_(0.25)
    check_search(c, p, q, table, lens, 4, cu)
