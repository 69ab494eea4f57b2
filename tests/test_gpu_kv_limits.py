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
