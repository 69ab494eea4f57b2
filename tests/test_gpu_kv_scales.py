"""KvCache.attend of prompts over 8 bits where the rows' scales are many powers of two apart: what a query does not see has no part
in its result, whichever queries share its tile."""
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
