"""The key/value cache as a model's layer uses it: prompts and then tokens added, searched and attended to, eagerly and captured."""
import pytest
import torch

from tests.kv_plain import PlainCache
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


class Layer:
    """One attention layer over random projections, with the cache under test."""

    def __init__(self, pages, heads, group, dim, page, dtype, kind, k):
        import ferrolm_b200 as fv

        self.c = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind=kind)
        self.heads, self.group, self.k = heads, group, k

    def step(self, rows, table, lens, cu=None):
        """(blocks, result, logarithms) of rows (n, heads * (group + 2), dim): queries, keys, values."""
        q, k, v = rows.split([self.heads * self.group, self.heads, self.heads], 1)
        self.c.add(k, v, table, lens, cu=cu)
        blocks = self.c.search_blocks(q, table, lens, self.k, cu=cu)
        return (blocks, *self.c.attend(q, table, lens, cu=cu, blocks=blocks, return_lse=True))


def rows_of(n, heads, group, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((n, heads * (group + 2), dim), generator=g).to(dtype)


@pytest.mark.parametrize("kind,dtype,heads,group,dim,page", [("same", BF, 2, 4, 64, 16), ("int8", FP, 1, 3, 96, 32), ("e4m3", BF, 2, 8, 128, 16)])
def test_prompts_and_tokens_against_the_plain_cache(kind, dtype, heads, group, dim, page):
    """Three prompts at once, one in two pieces, then tokens; every step compared with the plain cache that did the same."""
    k, B, width = 4, 3, 9
    layer, p = Layer(B * width + 2, heads, group, dim, page, dtype, kind, k), PlainCache(B * width + 2, heads, dim, page, dtype, kind)
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(B * width + 2, generator=g)[: B * width].view(B, width).to(torch.int32)
    lens = [0, 0, 0]
    for step, new in enumerate([[5 * page + 3, 2 * page, 40], [17, 0, 2 * page + 1], [1, 1, 1], [1, 1, 1], [2, 5, 1]]):
        lens = [a + b for a, b in zip(lens, new)]
        cu = None if new == [1, 1, 1] else i32([0, new[0], new[0] + new[1], sum(new)])
        rows = rows_of(sum(new), heads, group, dim, dtype, 10 + step)
        q, kk, v = rows.split([heads * group, heads, heads], 1)
        blocks, out, lse = layer.step(rows.cuda(), table.cuda(), i32(lens).cuda(), None if cu is None else cu.cuda())
        p.add(kk, v, table, lens, cu)
        want = p.search(q, table, lens, k, cu, 1, 2, torch.zeros((sum(new), heads, k), dtype=torch.int64))
        assert torch.equal(blocks.cpu().long(), want), step
        ref = p.attend(q, table, lens, cu, want, dim**-0.5, torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64))
        assert ((out.cpu().double() - ref[0]).abs() <= ref[2]).all() and ((lse.cpu().double() - ref[1]).abs() <= ref[3]).all(), step


def test_a_captured_step_is_the_eager_one():
    """A padded decoding step in a graph: replayed over growing sequences, with sequences of no rows behind the live ones."""
    heads, group, dim, page, k, B = 2, 4, 128, 64, 6, 8
    eager, captured = (Layer(200, heads, group, dim, page, BF, "int8", k) for _ in range(2))
    table = torch.randperm(200, generator=torch.Generator().manual_seed(3))[: B * 20].view(B, 20).to(torch.int32).cuda()
    lens, cu, rows = i32([0] * B).cuda(), i32([0] * (B + 1)).cuda(), rows_of(B, heads, group, dim, BF, 1).cuda()
    out, lse = torch.zeros((B, heads * group, dim), dtype=BF, device="cuda"), torch.zeros((B, heads * group), device="cuda")
    blocks = torch.zeros((B, heads, k), dtype=torch.int32, device="cuda")

    def step():
        q, kk, v = rows.split([heads * group, heads, heads], 1)
        captured.c.add(kk, v, table, lens, cu=cu)
        captured.c.search_blocks(q, table, lens, k, cu=cu, out=blocks)
        captured.c.attend(q, table, lens, cu=cu, blocks=blocks, return_lse=True, out=(out, lse))

    # the sequences' earlier rows, in both caches
    old = [700, 64, 1, 1200, 333]
    first = rows_of(sum(old), heads, group, dim, BF, 2).cuda()
    start = torch.cat((i32([0]), i32(old).cumsum(0).to(torch.int32))).cuda()
    for layer in (eager, captured):
        layer.step(first, table[:5], i32(old).cuda(), start)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(1, 5):
        live = 5 - n % 2  # of the eight places
        lens.copy_(i32([x + n for x in old] + [0] * 3))
        cu.copy_(i32(list(range(live + 1)) + [live] * (B - live)))
        rows.copy_(rows_of(B, heads, group, dim, BF, 20 + n))
        out.fill_(3.5), lse.fill_(3.5), blocks.fill_(-9)
        graph.replay()
        want = eager.step(rows[:live], table[:live], lens[:live])
        assert torch.equal(blocks[:live], want[0]) and torch.equal(out[:live], want[1]) and torch.equal(lse[:live], want[2])
        assert (out[live:] == 3.5).all() and (lse[live:] == 3.5).all() and (blocks[live:] == -9).all()
    for name in ("k", "v", "k_scale", "v_scale", "bounds", "bound_codes", "bound_scale"):
        # the fifth sequence's rows of the steps that it was left out of are not there: compared without its pages
        keep = torch.ones(200, dtype=torch.bool)
        keep[table[4].cpu().long()] = False
        assert torch.equal(getattr(eager.c, name)[keep.cuda()].float(), getattr(captured.c, name)[keep.cuda()].float()), name


def test_two_caches_on_two_streams():
    """Two layers' steps at the same time: nothing is shared between calls."""
    heads, group, dim, page, k = 4, 4, 128, 64, 8
    layers = [Layer(300, heads, group, dim, page, dtype, kind, k) for dtype, kind in ((BF, "same"), (FP, "e4m3"))]
    table, lens, new = torch.randperm(300)[:280].view(1, 280).to(torch.int32).cuda(), i32([17000]).cuda(), [17000, 1, 300, 1]
    rows = [[rows_of(n, heads, group, dim, layer.c.dtype, 5 + i).cuda() for i, n in enumerate(new)] for layer in layers]

    def run(layer, rows):
        got, n = [], 0
        for x in rows:
            n += len(x)
            got.append(layer.step(x, table, torch.full_like(lens, n), i32([0, len(x)]).cuda()))
        return got

    alone = [run(layer, x) for layer, x in zip(layers, rows)]
    for _ in range(3):
        streams, together = [torch.cuda.Stream() for _ in layers], []
        for layer, x, s in zip(layers, rows, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                together.append(run(layer, x))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for a, b in zip(alone, together):
            for x, y in zip(a, b):
                assert all(torch.equal(u, v) for u, v in zip(x, y))


def test_all_blocks_listed_are_the_whole_sequence():
    """With as many blocks as there are, a search finds all of them and attention over them is attention over everything."""
    heads, group, dim, page = 2, 2, 64, 32
    layer = Layer(60, heads, group, dim, page, FP, "same", 20)
    table = torch.randperm(60)[:40].view(2, 20).to(torch.int32).cuda()
    rows, lens = rows_of(900, heads, group, dim, FP, 1).cuda(), i32([500, 400]).cuda()
    blocks, out, lse = layer.step(rows, table, lens, i32([0, 500, 900]).cuda())
    pos = torch.cat((torch.arange(500), torch.arange(400)))
    want = torch.arange(20)[None, None].expand(900, heads, 20)
    assert torch.equal(blocks.cpu().long(), torch.where(want <= (pos // page)[:, None, None], want, -1))
    q = rows[:, : heads * group]
    whole = layer.c.attend(q, table, lens, cu=i32([0, 500, 900]).cuda(), return_lse=True)
    assert torch.equal(out, whole[0]) and torch.equal(lse, whole[1])
