"""Calls over caches without a page: nothing is seen, whatever the kind and however many rows a sequence brings."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_kv_rows import i32

KINDS = ["same", "int8", "e4m3", "int4x32"]


@pytest.mark.parametrize("rows,width,group", [(8, 12, 1), (30, 400, 4), (200, 90, 12), (9, 3, 1), (2000, 50, 3)])
def test_work_is_that_of_what_will_run(rows, width, group):
    """Without pages a call goes row by row, over any kind, and wants what single rows want."""
    from ferrolm_b200._lib import lib
    from tests.test_kv_cpu import AT, batch, cache

    b = batch(table_width=width, table_stride=width, cu=AT, nseq=1, rows=rows)
    of = lambda kind: lib().fv_kv_attend_work(C.byref(cache(kind=kind, heads=1, pages=0)), C.byref(b), group)  # noqa: E731
    tasks = rows * -(-group // (8 if group <= 8 else 16))
    assert of(4) == of(1)
    assert of(4) == 0 or of(4) >= tasks * (8 if group <= 8 else 16) * 130 * 4


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width,heads,group", [(8, 12, 1, 1), (1, 300, 2, 4), (200, 90, 2, 12), (5, 2000, 1, 3)])
def test_attention_over_no_pages(kind, rows, width, heads, group):
    import ferrolm_b200 as fv

    c = fv.KvCache(0, heads, 128, page_size=64, kind=kind)
    q = torch.randn((rows + 1, heads * group, 128)).bfloat16().cuda()
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device="cuda")
    c.attend(q, torch.zeros((1, width), dtype=torch.int32, device="cuda"), i32([width * 64]).cuda(), cu=i32([0, rows]).cuda(), return_lse=True, out=(out, lse))
    assert (out[:rows] == 0).all() and (lse[:rows] == -torch.inf).all() and (out[rows:] == 3).all() and (lse[rows:] == 3).all()
