"""Which entries two tables share, from their addresses alone, against sets."""
import ctypes as C
import random

import pytest
import torch

from tests.test_kv_cpu import ARG, AT, CUDA, fv  # noqa: F401
from tests.test_rotary_pages_cpu import pages


def entries(t):
    return {t.table + 4 * (i * t.stride + j) for i in range(t.nseq) for j in range(t.width)}


@pytest.mark.parametrize("seed", range(4))
def test_entries_that_two_tables_share(fv, seed):  # noqa: F811
    from ferrolm_b200._lib import fv_table
    from ferrolm_b200.pages import _shared

    r, met = random.Random(seed), 0
    for _ in range(3000):
        a, b = (fv_table(4096 + 4 * r.randint(0, 60), (s := r.randint(1, 12)), r.randint(0, s), r.randint(0, 6)) for _ in range(2))
        if r.random() < 0.5:
            b.stride = a.stride
            b.width = min(b.width, a.stride)
        if r.random() < 0.2:  # the stride of a single row is anything
            a.nseq, a.stride = 1, r.choice([0, 1, 3, 1000])
        both = len(entries(a) & entries(b))
        assert _shared(a, b) == both and _shared(b, a) == both, [(t.table, t.stride, t.width, t.nseq) for t in (a, b)]
        met += both > 0
    assert met > 500


def test_tables_that_are_part_of_others_count_once(fv):  # noqa: F811
    from ferrolm_b200._lib import fv_table

    t, rows, columns, other = fv_table(4096, 8, 8, 6), fv_table(4096 + 4 * 16, 8, 8, 2), fv_table(4096 + 4 * 2, 8, 3, 6), fv_table(40960, 8, 8, 6)
    again, empty, across = fv_table(4096, 8, 8, 6), fv_table(4096, 8, 0, 6), fv_table(4096 + 4 * 44, 8, 8, 2)
    once = fv.KvPages._once
    assert once([t, again]) in ([t], [again]) and once([rows, t, columns]) == [t] and once([other, t]) == [other, t]
    assert once([rows, columns.__class__(4096 + 4 * 32, 8, 3, 2)]) and once([t, empty, other]) == [t, other]
    assert once([t, again, rows, again, other, other]) in ([t, other], [again, other])
    for tables in ([t, across], [across, t], [rows, columns], [other, t, across]):
        with pytest.raises(fv.FerrovecError, match="share"):
            once(tables)
    assert once([across, t, fv_table(4096, 8, 8, 8)])[0].nseq == 8


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses would be followed")
@pytest.mark.parametrize("seed", range(3))
def test_forks_into_the_table_itself(fv, seed):  # noqa: F811
    """Refused where an entry lies in both; parts of one tensor that share none are not."""
    from ferrolm_b200._lib import fv_table

    L, r, met = fv.kv.lib(), random.Random(seed), 0
    for _ in range(2000):
        a, b = (fv_table(AT + 4 * r.randint(0, 60), (s := r.randint(1, 12)), r.randint(1, s), r.randint(1, 6)) for _ in range(2))
        if r.random() < 0.5:
            b.stride, b.width = a.stride, min(b.width, a.stride)
        if r.random() < 0.2:
            a.nseq, a.stride = 1, r.choice([0, 1, 3, 1 << 40])
        both = bool(entries(a) & entries(b))
        for x, y in ((a, b), (b, a)):
            status = L.fv_pages_fork_dev(C.byref(pages()), None, C.byref(x), AT, AT, C.byref(y))
            assert status == (ARG if both or a.table == b.table else CUDA), [(t.table, t.stride, t.width, t.nseq) for t in (a, b)]
        met += both
    assert met > 300
    far = fv_table(AT + 8, 1 << 40, 2, 1 << 20)  # of no memory that there is
    assert L.fv_pages_fork_dev(C.byref(pages()), None, C.byref(far), AT, AT, C.byref(fv_table(AT, 2, 2, 3))) == ARG
