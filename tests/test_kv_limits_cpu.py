"""What the key/value cache's entry points refuse because of its size, and what they say that a call needs; all before any CUDA call."""
import ctypes as C

from tests.test_kv_cpu import UNSUPPORTED, batch, cache, calls, fv  # noqa: F401


def test_a_table_whose_last_block_ends_behind_31_bits(fv):  # noqa: F811
    """16,777,216 blocks of 128 rows: the position behind the last row of the last one is 2^31.  One block less, or smaller ones, are fine."""
    for name, call in calls(fv).items():
        if name == "fv_kv_search_dev":  # takes 50,000
            continue
        assert call(cache(page_size=128), batch(table_width=1 << 24)) == UNSUPPORTED
        assert fv.kv.lib().fv_last_error().decode().startswith(name)
        for page, width in ((128, (1 << 24) - 1), (64, 1 << 24)):
            assert call(cache(page_size=page), batch(table_width=width, nseq=0, rows=0)) == 0


def test_only_calls_that_may_cut_their_work_ask_for_memory(fv):  # noqa: F811
    """Rows by themselves over a table that is long enough do; prompts, which go another way, and short tables do not."""
    def work(rows, nseq, width, group=4):
        return fv.kv.lib().fv_kv_attend_work(C.byref(cache()), batch(rows=rows, nseq=nseq, table_width=width, cu=1 << 20), group)

    assert work(4, 1, 300) > 0 and work(1, 1, 300) > 0 and work(8, 2, 300) > 0
    assert work(5, 1, 300) == work(200, 10, 300) == work(40, 1, 300, 128) == 0
    assert work(4, 1, 2) == 0
    assert work(40, 1, 20_000) > 0  # the whole table's list has no room there, so such rows may go by themselves
