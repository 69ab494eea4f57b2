"""Refusals of the entry points for rotary positions and pages, which come before any CUDA call; the addresses are never followed."""
import ctypes as C

import pytest
import torch

from tests.kv_plain_pages import PlainPages
from tests.test_kv_cpu import ARG, AT, CUDA, UNSUPPORTED, cache, fv  # noqa: F401


def rotary(**change):
    from ferrolm_b200._lib import fv_rotary

    return fv_rotary(**(dict(device=0, dtype=0, dim=128, part=64, layout=0, amplitude=1.0, turns=AT) | change))


def rows(**change):
    from ferrolm_b200._lib import fv_rotary_rows

    return fv_rotary_rows(**(dict(in_=AT, out=AT, in_row=1024, in_head=128, out_row=1024, out_head=128, heads=8) | change))


def rotate(fv, r=None, x=None, count=1, n=3, lens=AT, cu=None, nseq=3, positions=None):  # noqa: F811
    return fv.kv.lib().fv_rotate_dev(C.byref(r or rotary()), None, C.byref(x or rows()), count, n, lens, cu, nseq, positions, 0)


def test_turns_that_are_refused(fv):  # noqa: F811
    L = fv.kv.lib()
    for status, change in ((UNSUPPORTED, dict(dtype=2)), (UNSUPPORTED, dict(layout=2)), (UNSUPPORTED, dict(dim=0)), (UNSUPPORTED, dict(dim=72)), (UNSUPPORTED, dict(dim=1040)),
                           (UNSUPPORTED, dict(part=144)), (UNSUPPORTED, dict(part=24)), (UNSUPPORTED, dict(part=0)), (ARG, dict(device=-1)), (ARG, dict(turns=None)),
                           (ARG, dict(turns=AT + 4)), (ARG, dict(amplitude=float("nan"))), (ARG, dict(amplitude=float("inf")))):
        assert rotate(fv, r=rotary(**change)) == status, change
        assert L.fv_last_error().decode().startswith("fv_rotate_dev")
    for status, change in ((UNSUPPORTED, dict(heads=0)), (UNSUPPORTED, dict(heads=1 << 16)), (ARG, dict(in_=None)), (ARG, dict(out=None)), (ARG, dict(in_=AT + 8)), (ARG, dict(out=AT + 2)),
                           (ARG, dict(in_row=1028)), (ARG, dict(out_head=4))):
        assert rotate(fv, x=rows(**change)) == status, change
    for status, change in ((UNSUPPORTED, dict(count=0)), (UNSUPPORTED, dict(count=5)), (ARG, dict(n=4)), (ARG, dict(lens=None)), (ARG, dict(lens=AT + 1)), (ARG, dict(cu=AT + 2)),
                           (ARG, dict(positions=AT + 3)), (UNSUPPORTED, dict(n=1 << 31, cu=AT)), (UNSUPPORTED, dict(nseq=1 << 30, n=1 << 30))):
        assert rotate(fv, **change) == status, change
    assert L.fv_rotate_dev(None, None, C.byref(rows()), 1, 3, AT, None, 3, None, 0) == ARG
    assert L.fv_rotate_dev(C.byref(rotary()), None, None, 1, 3, AT, None, 3, None, 0) == ARG
    assert rotate(fv, n=0, nseq=0, lens=None) == 0
    if not torch.cuda.is_available():
        assert rotate(fv) == CUDA and "no CPU path" in L.fv_last_error().decode()


@pytest.mark.parametrize("change", [dict(dim=72), dict(part=144), dict(part=24), dict(layout="both"), dict(base=0.0), dict(factor=-1.0), dict(original=0), dict(fast=1.0, slow=2.0),
                                    dict(frequencies=[1.0] * 63), dict(frequencies=[float("nan")] * 64), dict(amplitude=float("inf")), dict(device="cpu")])
def test_turns_that_cannot_be_made(fv, change):  # noqa: F811
    with pytest.raises(fv.FerrovecError):
        fv.Rotary(**(dict(dim=128) | change))


def pages(**change):
    from ferrolm_b200._lib import fv_pages

    return fv_pages(**(dict(device=0, page_size=64, pages=10, refs=AT) | change))


def table(**change):
    from ferrolm_b200._lib import fv_table

    return fv_table(**(dict(table=AT, stride=4, width=4, nseq=3) | change))


def page_calls(fv):  # noqa: F811
    """name -> call(pages, table)."""
    L, big = fv.kv.lib(), 1 << 20
    one = lambda c: (C.c_void_p * 1)(C.addressof(c))  # noqa: E731
    c = cache()
    return {
        "fv_pages_fork_dev": lambda p, t: L.fv_pages_fork_dev(C.byref(p), None, C.byref(t), AT, AT, C.byref(table(table=2 * AT))),
        "fv_pages_free_dev": lambda p, t: L.fv_pages_free_dev(C.byref(p), None, C.byref(t), AT),
        "fv_pages_extend_dev": lambda p, t: L.fv_pages_extend_dev(C.byref(p), None, one(c), 1, C.byref(t), AT, AT, AT, AT, big),
        "fv_pages_remap_dev": lambda p, t: L.fv_pages_remap_dev(C.byref(p), None, AT, C.byref(t)),
    }


def test_pages_and_tables_that_are_refused(fv):  # noqa: F811
    L = fv.kv.lib()
    for name, call in page_calls(fv).items():
        for status, change in ((UNSUPPORTED, dict(page_size=48)), (UNSUPPORTED, dict(pages=1 << 31)), (ARG, dict(device=-1)), (ARG, dict(refs=None)), (ARG, dict(refs=AT + 2))):
            assert call(pages(**change), table()) == status, (name, change)
            assert L.fv_last_error().decode().startswith(name)
        for status, change in ((UNSUPPORTED, dict(nseq=1 << 30)), (UNSUPPORTED, dict(width=1 << 25, stride=1 << 25)), (ARG, dict(table=None)), (ARG, dict(table=AT + 1)), (ARG, dict(stride=3))):
            assert call(pages(), table(**change)) == status, (name, change)
        if not torch.cuda.is_available():
            assert call(pages(), table()) == CUDA, name
    assert L.fv_pages_fork_dev(C.byref(pages()), None, C.byref(table()), AT, None, C.byref(table(table=2 * AT))) == ARG
    assert L.fv_pages_fork_dev(C.byref(pages()), None, C.byref(table()), AT, AT, C.byref(table())) == ARG  # the table itself
    assert L.fv_pages_remap_dev(C.byref(pages()), None, None, C.byref(table())) == ARG


def test_caches_and_work_of_pages(fv):  # noqa: F811
    L = fv.kv.lib()
    for c in (cache(pages=11), cache(page_size=32), cache(device=1)):
        held = (C.c_void_p * 1)(C.addressof(c))
        assert L.fv_pages_extend_dev(C.byref(pages()), None, held, 1, C.byref(table()), AT, AT, AT, AT, 1 << 20) == ARG
        assert L.fv_pages_compact_dev(C.byref(pages()), None, held, 1, AT, AT, AT, 1 << 20) == ARG
    c = cache()
    held = (C.c_void_p * 1)(C.addressof(c))
    size = L.fv_pages_extend_work(C.byref(pages()), C.byref(table()))
    assert size >= 4 * (1 + 4 + 3 * 10)
    for work, n in ((None, size), (AT, size - 1), (AT + 8, size)):
        assert L.fv_pages_extend_dev(C.byref(pages()), None, held, 1, C.byref(table()), AT, AT, AT, work, n) == ARG
    size = L.fv_pages_compact_work(C.byref(pages()))
    for work, n in ((None, size), (AT, size - 1), (AT + 4, size)):
        assert L.fv_pages_compact_dev(C.byref(pages()), None, held, 1, AT, AT, work, n) == ARG
    assert L.fv_pages_compact_dev(C.byref(pages()), None, held, 1, None, AT, AT, size) == ARG
    assert L.fv_pages_extend_dev(C.byref(pages()), None, held, 1, C.byref(table()), None, AT, AT, AT, 1 << 20) == ARG
    assert L.fv_pages_extend_dev(C.byref(pages()), None, held, 1, C.byref(table()), AT, AT, None, AT, 1 << 20) == ARG


def test_copies_that_are_refused(fv):  # noqa: F811
    L = fv.kv.lib()
    for kind in (0, 1, 2, 4):
        c = cache(kind=kind)
        assert L.fv_kv_copy_pages_dev(C.byref(c), None, None, AT, 3, None) == ARG
        assert L.fv_kv_copy_pages_dev(C.byref(c), None, AT, AT + 2, 3, None) == ARG
        assert L.fv_kv_copy_pages_dev(C.byref(c), None, AT, AT, 3, AT + 1) == ARG
        assert L.fv_kv_copy_pages_dev(C.byref(c), None, AT, AT, 1 << 32, None) == UNSUPPORTED
        assert L.fv_kv_copy_pages_dev(C.byref(c), None, None, None, 0, None) == 0
    assert L.fv_kv_copy_pages_dev(C.byref(cache(kind=3)), None, AT, AT, 3, None) == UNSUPPORTED


def test_plain_pages():
    """The plain form itself, on a case worked out by hand: three beams of one sequence of 20 rows, two of which go on."""
    p = PlainPages(9, 16)
    table = [[-1] * 3]
    p.extend(table, [0], [20])
    assert table == [[0, 1, -1]] and p.refs[:3] == [1, 1, 0]
    kids = p.fork(table, [20], [0, 0, 0])
    assert p.refs[:2] == [4, 4]
    p.free(table)
    p.extend(kids, [20] * 3, [1, 1, -1])  # the third holds page 1 as well and is left as it is
    assert kids == [[0, 2, -1], [0, 3, -1], [0, 1, -1]] and p.refs[:4] == [3, 1, 1, 1] and p.copied == [(1, 2), (1, 3)]
    p.extend(kids, [21, 21, 20], [1, 1, 12])
    assert kids == [[0, 2, -1], [0, 3, -1], [0, 1, -1]]
    p.free(kids, [0, 21, 0])
    p.compact(kids)
    assert kids == [[-1] * 3, [0, 1, -1], [-1] * 3] and p.refs[:3] == [1, 1, 0]
