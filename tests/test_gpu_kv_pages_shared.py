"""KvPages where tables share memory with one another, and with more caches than one launch copies."""
import pytest
import torch

from tests.test_gpu_kv_pages import ALL, bits, make, moved, same, same_rows
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu


def half_used(pages, page, layers, table):
    """Every second of the pages that `table` names is in use, once for each of its rows that has it."""
    caches, p, plain = make(pages, page, layers)
    d = table.cuda()
    for q in range(pages):
        plain.refs[q] = int((table == q).sum()) if q % 2 else 0
    p.refs.copy_(i32(plain.refs))
    return caches, p, plain, d


TABLE = torch.tensor([[9, 1, -1, 19], [7, 5, 13, 0], [15, 11, 3, 40], [17, 1, 4, -7]], dtype=torch.int32)


@pytest.mark.parametrize("which", ["twice", "a view first", "a view last", "columns", "rows between", "views that meet nowhere", "three times"])
def test_an_entry_is_renumbered_once(which):
    """A table given twice, or with views of itself, is as if it were given once."""
    caches, p, plain, t = half_used(20, 16, ALL, TABLE)
    want, rows = TABLE.tolist(), bits(caches)
    p.compact(*{"twice": (t, t), "a view first": (t[1:3], t), "a view last": (t, t[:2]), "columns": (t, t[:, 1:3]), "rows between": (t[::2], t, t[1::2]),
                "views that meet nowhere": (t[:, :1], t[:2, 1:], t[2:, 1:]), "three times": (t, t.view(4, 4), t)}[which])
    plain.compact(want)
    assert plain.copied
    same(t, p, want, plain)
    same_rows(caches, moved(rows, plain.copied))


def test_pages_that_nobody_holds_are_none_in_the_end():
    """An entry that names a free page becomes -1, also where another page moves to that place."""
    _, p, _, t = half_used(6, 16, ALL[:1], i32([[1, 3, 5, 0, 2, 4]]))
    p.compact(t, t)
    assert t.tolist() == [[1, 0, 2, -1, -1, -1]]


@pytest.mark.parametrize("views", [lambda t: (t[:3], t[2:]), lambda t: (t[:, :3], t[:, 2:]), lambda t: (t[:3, :3], t[1:, 1:]), lambda t: (t[::2], t[1:3])])
def test_tables_that_share_some_entries_are_refused(views):
    """Before anything moves."""
    import ferrolm_b200 as fv

    caches, p, plain, t = half_used(20, 16, ALL[:1], TABLE)
    rows = bits(caches)
    with pytest.raises(fv.FerrovecError, match="share"):
        p.compact(*views(t))
    same(t, p, TABLE.tolist(), plain)
    same_rows(caches, rows)
    assert int(p.used) == 0


def test_a_table_that_cannot_be_renumbered_is_refused_before_anything_moves():
    import ferrolm_b200 as fv

    caches, p, plain, t = half_used(20, 16, ALL[:1], TABLE)
    rows, wide = bits(caches), torch.full((1, (1 << 24) + 1), 1, dtype=torch.int32, device="cuda")
    with pytest.raises(fv.FerrovecError):
        p.compact(t, wide)
    same(t, p, TABLE.tolist(), plain)
    same_rows(caches, rows)
    assert int(p.used) == 0 and int(wide.min()) == 1


def test_forks_into_the_table_itself_are_refused():
    """Threads would read what others write.  Other parts of the same tensor are fine."""
    import ferrolm_b200 as fv

    _, p, plain, t = half_used(20, 16, ALL[:1], TABLE.repeat(2, 1))
    n, parents = i32([64] * 4).cuda(), i32([3, 0, 1]).cuda()
    for out in (t[1:4], t[:3], t[3:6], t[2:5, 1:]):
        with pytest.raises(fv.FerrovecError, match="shares"):
            p.fork(t[:4], n, parents, out=out)
    assert torch.equal(t.cpu(), TABLE.repeat(2, 1)) and p.refs.tolist() == plain.refs
    p.fork(t[:4], n, parents, out=t[4:7])
    assert t[4:7].tolist() == plain.fork(TABLE.tolist(), [64] * 4, [3, 0, 1]) and torch.equal(t[:4].cpu(), TABLE)
    assert p.refs.tolist() == plain.refs
    p.fork(t[:3, :2], n[:3], parents[1:], out=t[:2, 2:])
    assert t[:2, 2:].tolist() == plain.fork([r[:2] for r in TABLE.tolist()], [64] * 4, [0, 1])


@pytest.mark.parametrize("layers", [8, 9, 16, 33])
def test_many_caches(layers):
    """More caches than one launch copies: every one has what the first has, and counts move once."""
    caches, p, plain = make(60, 16, tuple(ALL[i % len(ALL)] for i in range(layers)), layers)
    table, want = torch.full((4, 6), -1, dtype=torch.int32, device="cuda"), [[-1] * 6 for _ in range(4)]
    lens, zero = [40, 17, 90, 3], [0] * 4
    p.extend(table, i32(zero).cuda(), i32(lens).cuda()), plain.extend(want, zero, lens)
    for step in range(3):
        parents = [[0, 0, 1, 2], [3, 3, 3, 0], [2, 1, 1, 3]][step]
        kids, theirs = p.fork(table, i32(lens).cuda(), i32(parents).cuda()), plain.fork(want, lens, parents)
        lens, rows = [lens[b] for b in parents], bits(caches)
        p.extend(kids, i32(lens).cuda(), i32([1, 20, 0, 5]).cuda()), plain.extend(theirs, lens, [1, 20, 0, 5])
        assert plain.copied and int(p.missing) == plain.missing == 0
        same(kids, p, theirs, plain)
        same_rows(caches, moved(rows, plain.copied))
        p.free(table), plain.free(want)
        rows = bits(caches)
        p.compact(kids), plain.compact(theirs)
        same(kids, p, theirs, plain)
        same_rows(caches, moved(rows, plain.copied))
        table, want, lens = kids, theirs, [a + b for a, b in zip(lens, [1, 20, 0, 5])]
        lens = [min(n, 96) for n in lens]
