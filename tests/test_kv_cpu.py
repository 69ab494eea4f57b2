"""Refusals of the key/value cache's entry points.  They come before any CUDA call, so they are the same without a GPU; the
addresses that the calls get here are never followed."""
import ctypes as C

import pytest
import torch

ARG, CUDA, UNSUPPORTED = 1, 3, 6
AT = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def fv():
    import __graft_entry__ as g

    g.build()
    import ferrolm_b200

    return ferrolm_b200


def cache(kind=1, **change):
    from ferrolm_b200._lib import fv_kv

    scale = AT if kind else None
    c = dict(device=0, dtype=0, kind=kind, page_size=64, heads=8, dim=128, pages=10, k=AT, v=AT, k_scale=scale, v_scale=scale, bounds=AT,
             bound_codes=AT, bound_scale=AT)
    return fv_kv(**(c | change))


def batch(**change):
    from ferrolm_b200._lib import fv_kv_batch

    return fv_kv_batch(**(dict(table=AT, table_stride=4, table_width=4, lens=AT, cu=None, nseq=3, rows=3) | change))


def calls(fv):
    """name -> call(cache, batch) with arguments of its own that are fine."""
    L = fv.kv.lib()
    return {
        "fv_kv_add_dev": lambda c, b: L.fv_kv_add_dev(C.byref(c), None, C.byref(b), AT, 1024, 128, AT, 1024, 128),
        "fv_kv_vectors_dev": lambda c, b: L.fv_kv_vectors_dev(C.byref(c), None, C.byref(b), AT, AT),
        "fv_kv_search_dev": lambda c, b: L.fv_kv_search_dev(C.byref(c), None, C.byref(b), AT, 4096, 128, 4, 8, 1, 2, AT),
        "fv_kv_attend_dev": lambda c, b: L.fv_kv_attend_dev(C.byref(c), None, C.byref(b), AT, 4096, 128, 4, AT, 8, 0.1, AT, AT, None, 0),
    }


BAD = [
    (UNSUPPORTED, dict(dtype=2), {}), (UNSUPPORTED, dict(kind=3), {}), (UNSUPPORTED, dict(kind=-1), {}), (UNSUPPORTED, dict(dim=80), {}),
    (UNSUPPORTED, dict(dim=0), {}), (UNSUPPORTED, dict(page_size=48), {}), (UNSUPPORTED, dict(page_size=256), {}), (UNSUPPORTED, dict(heads=0), {}),
    (UNSUPPORTED, dict(heads=1 << 16), {}), (UNSUPPORTED, dict(pages=1 << 31), {}), (ARG, dict(device=-1), {}), (ARG, dict(k=None), {}),
    (ARG, dict(v_scale=None), {}), (ARG, dict(bounds=None), {}), (ARG, dict(bound_scale=None), {}), (ARG, dict(v=AT + 8), {}),
    (ARG, dict(bound_codes=AT + 4), {}), (ARG, dict(k_scale=AT + 2), {}), (ARG, {}, dict(lens=None)), (ARG, {}, dict(table=None)),
    (ARG, {}, dict(rows=4)), (ARG, {}, dict(lens=AT + 1)), (ARG, {}, dict(cu=AT + 2)), (UNSUPPORTED, {}, dict(rows=1 << 31, cu=AT)),
    (UNSUPPORTED, {}, dict(nseq=1 << 30, rows=1 << 30)), (UNSUPPORTED, {}, dict(table_width=1 << 25)),
]


@pytest.mark.parametrize("status,bad_cache,bad_batch", BAD)
def test_caches_and_batches_that_are_refused(fv, status, bad_cache, bad_batch):
    for name, call in calls(fv).items():
        assert call(cache(**bad_cache), batch(**bad_batch)) == status, name
        assert fv.kv.lib().fv_last_error().decode().startswith(name)


def test_a_cache_of_16_bits_has_no_scales(fv):
    for call in calls(fv).values():
        assert call(cache(kind=0, k_scale=AT), batch()) == ARG


def test_null_arguments(fv):
    L = fv.kv.lib()
    c, b = cache(), batch()
    assert L.fv_kv_add_dev(None, None, C.byref(b), AT, 1024, 128, AT, 1024, 128) == ARG
    assert L.fv_kv_add_dev(C.byref(c), None, None, AT, 1024, 128, AT, 1024, 128) == ARG
    assert L.fv_kv_add_dev(C.byref(c), None, C.byref(b), None, 1024, 128, AT, 1024, 128) == ARG
    assert L.fv_kv_add_dev(C.byref(c), None, C.byref(b), AT, 1024, 128, AT + 8, 1024, 128) == ARG
    assert L.fv_kv_add_dev(C.byref(c), None, C.byref(b), AT, 1024, 132, AT, 1024, 128) == ARG
    assert L.fv_kv_vectors_dev(C.byref(c), None, C.byref(b), AT, None) == ARG
    assert L.fv_kv_vectors_dev(C.byref(c), None, C.byref(b), AT + 2, AT) == ARG


def test_searches_that_are_refused(fv):
    L, c, b = fv.kv.lib(), cache(), batch()

    def search(q=AT, row=4096, head=128, group=4, k=8, first=1, recent=2, out=AT, batch=b):
        return L.fv_kv_search_dev(C.byref(c), None, C.byref(batch), q, row, head, group, k, first, recent, out)

    assert search(group=0) == search(group=129) == search(k=0) == search(k=4097) == UNSUPPORTED
    assert search(batch=batch(table_width=50001)) == UNSUPPORTED
    assert search(q=None) == search(out=None) == search(q=AT + 8) == search(row=4100) == search(head=4) == search(out=AT + 2) == ARG


def test_attentions_that_are_refused(fv):
    L, c, b = fv.kv.lib(), cache(), batch()

    def attend(q=AT, row=4096, head=128, group=4, blocks=AT, k=8, scale=0.1, out=AT, lse=AT, work=None, size=0):
        return L.fv_kv_attend_dev(C.byref(c), None, C.byref(b), q, row, head, group, blocks, k, scale, out, lse, work, size)

    assert attend(group=0) == attend(group=129) == attend(k=0) == attend(k=4097) == UNSUPPORTED
    assert attend(scale=float("nan")) == attend(scale=float("inf")) == ARG
    assert attend(q=None) == attend(out=None) == attend(q=AT + 8) == attend(row=4100) == attend(head=4) == ARG
    assert attend(out=AT + 8) == attend(lse=AT + 2) == attend(blocks=AT + 1) == attend(work=AT + 8) == ARG


def test_nothing_to_do_is_no_error(fv):
    for call in calls(fv).values():
        assert call(cache(), batch(nseq=0, rows=0, table=None, lens=None)) == 0
        assert call(cache(pages=0), batch(nseq=0, rows=0)) == 0


def test_rows_of_a_cache_without_pages(fv):
    for name in ("fv_kv_add_dev", "fv_kv_vectors_dev"):
        call = calls(fv)[name]
        assert call(cache(pages=0, k=None, v=None, k_scale=None, v_scale=None, bounds=None, bound_codes=None, bound_scale=None), batch()) == 0


def test_no_gpu_means_a_loud_failure(fv):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call in calls(fv).values():
        assert call(cache(), batch()) == CUDA
        assert "no CPU path" in fv.kv.lib().fv_last_error().decode()


@pytest.mark.parametrize("change", [dict(kind="int4"), dict(dtype=torch.float32), dict(dim=100), dict(page_size=8), dict(heads=0), dict(pages=-1)])
def test_caches_that_cannot_be_made(fv, change):
    with pytest.raises(fv.FerrovecError):
        fv.KvCache(**(dict(pages=4, heads=2, dim=64, page_size=16) | change))


def test_buffers_that_do_not_fit(fv):
    good = dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), v=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16),
                bounds=torch.zeros(4, 2, 2, 64, dtype=torch.bfloat16), bound_codes=torch.zeros(4, 2, 2, 64, dtype=torch.int8),
                bound_scale=torch.zeros(4, 2))
    with pytest.raises(fv.FerrovecError, match="CUDA device"):  # there is no CPU path
        fv.KvCache(4, 2, 64, page_size=16, buffers=good)
    for name, x in (("k", good["k"].half()), ("v", good["v"][:3]), ("bounds", good["bounds"].transpose(0, 1)), ("bound_scale", None)):
        with pytest.raises(fv.FerrovecError, match=name):
            fv.KvCache(4, 2, 64, page_size=16, buffers=good | {name: x})
    with pytest.raises(fv.FerrovecError, match="k_scale|buffers"):
        fv.KvCache(4, 2, 64, page_size=16, kind="int8", buffers=good)
