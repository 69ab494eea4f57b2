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
