"""KvPages against tests/kv_plain_pages.py: everything is a whole number or a copy, and compared exactly."""
import pytest
import torch

from tests.kv_plain_pages import PlainPages
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
BUFFERS = ("k", "v", "bounds", "bound_codes", "bound_scale", "k_scale", "v_scale")


def make(pages, page, layers=((2, 64, BF, "same"),), seed=0):
    """Caches full of random bits, their pages, and the plain ones."""
    import ferrolm_b200 as fv

    g = torch.Generator().manual_seed(seed)
    caches = [fv.KvCache(pages, h, d, page_size=page, dtype=t, kind=kind) for h, d, t, kind in layers]
    for c in caches:
        for name in BUFFERS:
            x = getattr(c, name)
            if x is not None:
                x.view(torch.uint8).copy_(torch.randint(0, 100, x.view(torch.uint8).shape, generator=g, dtype=torch.uint8))
    return caches, fv.KvPages(caches), PlainPages(pages, page)


def bits(caches):
    return [[None if getattr(c, n) is None else getattr(c, n).view(torch.uint8).flatten(1).cpu().clone() for n in BUFFERS] for c in caches]


def moved(before, copied):
    for layer in before:
        for x in layer:
            if x is not None and copied:
                src, dst = torch.tensor(copied).T
                x[dst] = x[src]
    return before


def same(table, pages, want, plain):
    assert table.tolist() == want and pages.refs.tolist() == plain.refs


def same_rows(caches, want):
    for a, b in zip(bits(caches), want):
        for x, y in zip(a, b):
            assert (x is None) == (y is None) and (x is None or torch.equal(x, y))


ALL = ((2, 64, BF, "same"), (3, 96, FP, "int8"), (1, 128, BF, "e4m3"), (5, 96, BF, "int4x32"), (7, 128, FP, "int4x32"))


@pytest.mark.parametrize("page,layers", [(16, ALL), (128, ALL[:2]), (64, (ALL[3],)), (32, ((40, 128, BF, "same"),))])
def test_copies(page, layers):
    """Every buffer of every kind, pages of more than one slice, pairs that are skipped."""
    caches, _, _ = make(30, page, layers)
    src, dst = [3, 29, 0, -1, 7, 30, 12], [4, 1, 28, 5, 2, 6, -3]
    want = moved(bits(caches), [(a, b) for a, b in zip(src, dst) if 0 <= a < 30 and 0 <= b < 30])
    for c in caches:
        c.copy_pages(i32(src).cuda(), i32(dst).cuda())
        c.copy_pages(i32([]).cuda(), i32([]).cuda())
    same_rows(caches, want)


def test_copies_of_scales_that_begin_on_4_bytes():
    import ferrolm_b200 as fv

    (c,), _, _ = make(9, 16, ((2, 64, BF, "int8"),))
    held = {n: getattr(c, n) for n in BUFFERS}
    room = torch.zeros(9 * 2 * 16 + 1, device="cuda")
    held["k_scale"] = room[1:].view(9, 2, 16).copy_(held["k_scale"])
    c = fv.KvCache(9, 2, 64, page_size=16, kind="int8", buffers=held)
    want = moved(bits([c]), [(2, 5), (0, 8)])
    c.copy_pages(i32([2, 0]).cuda(), i32([5, 8]).cuda())
    same_rows([c], want)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("B,width,pages", [(1, 1, 3), (5, 7, 60), (70, 40, 4000), (2100, 3, 9000), (3, 1500, 5001)])
def test_room(B, width, pages, page):
    """Lengths from nothing to the table's end and behind it, rows that stay in their block, cross one border or many."""
    g = torch.Generator().manual_seed(B)
    caches, p, plain = make(pages, page, ((1, 64, BF, "same"),))
    used = torch.randperm(pages, generator=g)[: pages // 5]
    p.refs[used.cuda()] = 1
    plain.refs = p.refs.tolist()
    lens, table = [0] * B, torch.full((B, width), -1, dtype=torch.int32)
    table[0, 0] = pages + 7  # no page
    want, d = table.tolist(), table.cuda()
    for step in range(4):
        more = torch.randint(-2, max(3, width * page // 3), (B,), generator=g).tolist()
        if step == 1:
            more = [1] * B
        p.extend(d, i32(lens).cuda(), i32(more).cuda())
        plain.extend(want, lens, more)
        assert int(p.missing) == plain.missing
        same(d, p, want, plain)
        p.extend(d, i32(lens).cuda(), i32(more).cuda())  # room that is there stays
        same(d, p, want, plain)
        lens = [n + max(m, 0) for n, m in zip(lens, more)]


@pytest.mark.parametrize("layers", [ALL, ALL[:1]])
@pytest.mark.parametrize("seed", range(4))
def test_sequences_that_share_pages(seed, layers):
    """Steps of sequences that go on from one another: some pages are held by sequences of the call alone, some by others too."""
    g = torch.Generator().manual_seed(seed)
    page, pages, width, B = 16, 400, 9, 12
    caches, p, plain = make(pages, page, layers, seed)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    want, lens = table.tolist(), [0] * B
    held, kept = [], []  # tables that are kept beside
    for step in range(8):
        more = torch.randint(0, 25, (B,), generator=g).tolist()
        rows = bits(caches)
        p.extend(table, i32(lens).cuda(), i32(more).cuda())
        plain.extend(want, lens, more)
        assert int(p.missing) == plain.missing == 0
        same(table, p, want, plain)
        same_rows(caches, moved(rows, plain.copied))
        lens = [min(n + m, width * page) for n, m in zip(lens, more)]
        parents = torch.randint(-1, B + 1, (B,), generator=g).tolist()
        children = p.fork(table, i32(lens).cuda(), i32(parents).cuda())
        theirs = plain.fork(want, lens, parents)
        same(children, p, theirs, plain)
        if step % 3 == 2:
            held.append(table), kept.append(want)
        else:
            p.free(table), plain.free(want)
            same(table, p, want, plain)
        table, want, lens = children, theirs, [lens[b] if 0 <= b < B else 0 for b in parents]
        cut = [max(0, n - int(torch.randint(0, 20, (1,), generator=g))) for n in lens]
        p.free(table, i32(cut).cuda()), plain.free(want, cut)
        same(table, p, want, plain)
        lens = cut
        if step % 2:
            rows = bits(caches)
            p.compact(table, *held), plain.compact(want, *kept)
            assert int(p.used) == plain.used
            same(table, p, want, plain)
            same_rows(caches, moved(rows, plain.copied))
            assert [x.tolist() for x in held] == kept
    for x, y in zip([table, *held], [want, *kept]):
        p.free(x), plain.free(y)
    same(table, p, want, plain)
    assert int(p.refs.sum()) == 0


@pytest.mark.parametrize("more", [[0, 0, 0], [0, -1, 0], [-1, -1, 5], [0, 3, -7]])
def test_begun_blocks_where_no_rows_come(more):
    """A begun block that is shared becomes the sequence's own with `more` 0 too; with less the sequence is left alone."""
    caches, p, plain = make(20, 16, ALL[2:4])
    table = torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
    p.extend(table, i32([0]).cuda(), i32([32]).cuda())
    want = [[-1] * 3]
    plain.extend(want, [0], [32])
    for lens in ([20, 20, 17], [32, 20, 16], [16, 31, 0]):
        kids, theirs = p.fork(table, None, i32([0, 0, 0]).cuda()), plain.fork(want, None, [0, 0, 0])
        rows = bits(caches)
        p.extend(kids, i32(lens).cuda(), i32(more).cuda()), plain.extend(theirs, lens, more)
        same(kids, p, theirs, plain)
        same_rows(caches, moved(rows, plain.copied))
        p.free(kids), plain.free(theirs)


def test_too_few_pages_change_nothing():
    caches, p, plain = make(6, 16)
    table = i32([[0, -1, -1], [0, -1, -1], [-9, -1, -1]]).cuda()
    p.refs.copy_(i32([2, 0, 1, 1, 0, 1]))
    plain.refs, want = p.refs.tolist(), table.tolist()
    rows = bits(caches)
    for lens, more, short in (([5, 7, 0], [1, 20, 40], 3), ([5, 7, 0], [1, 1, 32], 1)):  # free: 1 and 4
        p.extend(table, i32(lens).cuda(), i32(more).cuda()), plain.extend(want, lens, more)
        assert int(p.missing) == plain.missing == short
        same(table, p, want, plain)
    p.extend(table, i32([5, 7, 0]).cuda(), i32([1, 1, 3]).cuda()), plain.extend(want, [5, 7, 0], [1, 1, 3])
    assert int(p.missing) == 0 and plain.copied == [(0, 1)]
    same(table, p, want, plain)
    same_rows(caches, moved(rows, plain.copied))


@pytest.mark.parametrize("pages,live", [(1, 0), (1, 1), (127, 60), (128, 128), (4097, 1), (5000, 2500), (5000, 4990), (32768, 20000), (32769, 32768), (40001, 15000), (40001, 36000), (150000, 65536), (150000, 100000), (150000, 300), (131072, 131072)])
def test_compaction(pages, live):
    g = torch.Generator().manual_seed(pages + live)
    caches, p, plain = make(pages, 16, ((1, 64, BF, "int4x32"),))
    p.refs[torch.randperm(pages, generator=g)[:live].cuda()] = torch.randint(1, 5, (live,), generator=g, dtype=torch.int32).cuda()
    plain.refs = p.refs.tolist()
    table = torch.randint(-3, pages + 2, (5, 300), generator=g).to(torch.int32).cuda()
    want, rows = table.tolist(), bits(caches)
    p.compact(table), plain.compact(want)
    assert int(p.used) == live
    same(table, p, want, plain)
    same_rows(caches, moved(rows, plain.copied))
    p.compact(), p.compact(table[:0])
    same(table, p, want, plain)


@pytest.mark.parametrize("free", [[100_000, 7], [32_767, 32_768, 65_535, 65_536, 99_999], [99_998]])
def test_room_far_behind(free):
    """Free pages in windows behind the first, and fewer of them than are wanted."""
    caches, p, plain = make(100_001, 16, ((1, 64, BF, "int4x32"),))
    p.refs.fill_(1)
    p.refs[torch.tensor(free).cuda()] = 0
    plain.refs = p.refs.tolist()
    table, want = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), [[-1] * 4 for _ in range(3)]
    for more in ([17, 0, 0], [17, 1, 30], [40, 40, 40]):
        p.extend(table, i32([0, 0, 0]).cuda(), i32(more).cuda()), plain.extend(want, [0, 0, 0], more)
        assert int(p.missing) == plain.missing
        same(table, p, want, plain)


def test_tables_that_are_parts_of_others():
    """Strided tables, a fork to a wider one, one without lengths, a page given back more often than it is held."""
    _, p, plain = make(50, 32)
    wide = torch.full((4, 20), -1, dtype=torch.int32, device="cuda")
    part = wide[:, 3:10]
    p.extend(part, i32([0, 40, 0, 0]).cuda(), i32([100, 30, 0, 1000]).cuda())
    want = [[-1] * 7 for _ in range(4)]
    plain.extend(want, [0, 40, 0, 0], [100, 30, 0, 1000])
    same(part, p, want, plain)
    assert (wide[:, :3] == -1).all() and (wide[:, 10:] == -1).all()
    out = torch.full((3, 12), 7, dtype=torch.int32, device="cuda")
    assert p.fork(part, None, i32([3, 0, 0]).cuda(), out=out[:, 1:11]).data_ptr() == out[:, 1:].data_ptr()
    same(out[:, 1:11], p, plain.fork(want, None, [3, 0, 0], 10), plain)
    assert (out[:, 0] == 7).all() and (out[:, 11] == 7).all()
    again = part.clone()
    for _ in range(4):
        p.free(again.copy_(part)), plain.free([list(r) for r in want])
    assert p.refs.tolist() == plain.refs


def test_rows_stay_readable():
    """Rows added through a table are the same rows after a fork, an extension of both and a compaction."""
    import ferrolm_b200 as fv

    c = fv.KvCache(64, 2, 128, page_size=16, kind="int4x32")
    p = fv.KvPages(c)
    table, lens = torch.full((2, 6), -1, dtype=torch.int32, device="cuda"), i32([0, 0]).cuda()
    new, cu = i32([50, 30]).cuda(), i32([0, 50, 80]).cuda()
    p.refs[:9] = 1  # of somebody else
    p.extend(table, lens, new)
    k = torch.randn((80, 2, 128)).to(BF).cuda()
    c.add(k, -k, table, new, cu=cu)
    before = c.vectors(table, new, cu=cu, rows=80)
    both = p.fork(table, new, i32([0, 0, 1]).cuda())
    p.free(table)
    lens = new[[0, 0, 1]]
    p.extend(both, lens, i32([1, 1, 1]).cuda())
    x = torch.randn((3, 2, 128)).to(BF).cuda()
    c.add(x, x, both, lens + 1)
    p.refs[:9] = 0
    p.compact(both)
    assert int(p.used) == 3 + 2 + 2 and int(both.max()) == 6  # three whole pages shared, two begun ones of one page's rows, two of the other sequence
    got = c.vectors(both, lens, cu=i32([0, 50, 100, 130]).cuda(), rows=130)
    for a, b in zip(got, before):
        assert torch.equal(a, torch.cat((b[:50], b[:50], b[50:])))
    last = c.vectors(both, lens + 1)[0]
    assert last.isfinite().all() and not torch.equal(last[0], last[1])


def test_captured():
    """A step of beams in a graph: fork, give back, room."""
    _, p, plain = make(90, 16)
    table, lens = torch.full((4, 8), -1, dtype=torch.int32, device="cuda"), i32([3, 20, 15, 16]).cuda()
    parents, more, kids = i32([0, 0, 2, 1]).cuda(), i32([1] * 4).cuda(), torch.empty((4, 8), dtype=torch.int32, device="cuda")
    want = table.tolist()
    p.extend(table, torch.zeros_like(lens), lens), plain.extend(want, [0] * 4, [3, 20, 15, 16])

    def step():
        p.fork(table, lens, parents, out=kids)
        p.free(table)
        grown = lens[parents.long()]
        p.extend(kids, grown, more)
        table.copy_(kids)
        lens.copy_(grown + 1)

    keep = table.clone(), lens.clone(), p.refs.clone()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    table.copy_(keep[0]), lens.copy_(keep[1]), p.refs.copy_(keep[2])
    at, of = keep[1].tolist(), [0, 0, 2, 1]
    for n in range(20):
        graph.replay()
        theirs = plain.fork(want, at, of)
        plain.free(want)
        want, at = theirs, [at[b] for b in of]
        plain.extend(want, at, [1] * 4)
        at = [x + 1 for x in at]
        same(table, p, want, plain)


def test_refusals():
    import ferrolm_b200 as fv

    caches, p, _ = make(8, 16)
    t, n = torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), i32([1, 2]).cuda()
    for call in (lambda: p.extend(t.long(), n, n), lambda: p.extend(t, n[:1], n), lambda: p.extend(t, n, n.long()), lambda: p.extend(t[0], n, n),
                 lambda: p.extend(t.cpu(), n, n), lambda: p.extend(t[:, ::2], n, n), lambda: p.extend(t[:1].expand(2, 3), n, n), lambda: p.fork(t, n, n.long()),
                 lambda: p.fork(t, n, n, out=t), lambda: p.fork(t, n, n, out=t[:1]), lambda: p.fork(t, n[:1], n), lambda: p.free(t, n.float()), lambda: p.compact(t.t()),
                 lambda: caches[0].copy_pages(n, n[:1]), lambda: caches[0].copy_pages(n.long(), n), lambda: fv.KvPages([]), lambda: fv.KvPages([t]),
                 lambda: fv.KvPages([caches[0], fv.KvCache(9, 2, 64, page_size=16)]), lambda: fv.KvPages(caches, refs=n)):
        with pytest.raises(fv.FerrovecError):
            call()
