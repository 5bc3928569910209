"""CPU tests of the drafted-token operators' limits: calls at the edge of what a launch holds, outputs in what they read."""

import pytest

import pa_amd
from test_drafts import attend, keep, read
from test_new_tokens import A, BAD, LONG, message, rows


def test_keep_rows_at_its_limit():
    """2^20 entries of 32 heads are 2^25 items: 2^32 threads in a block-scaled cache, which no launch has."""
    assert keep(num_entries=1 << 20, num_kv_heads=32) == LONG and "2^25 - 1" in message()
    for dtype in (pa_amd.FP16, pa_amd.FP8_E4M3, pa_amd.FP8_E4M3_BLOCK):
        assert keep(dtype=dtype, num_entries=1 << 20, num_kv_heads=33, page_size=8) == LONG and "2^25" in message()
    # One entry fewer passes the check, and so does the limit elsewhere (refused only for the missing pointer behind it).
    assert keep(num_entries=(1 << 20) - 1, num_kv_heads=32, kept=None) != LONG and "null" in message()
    for dtype in (pa_amd.FP16, pa_amd.FP8_E4M3):
        assert keep(dtype=dtype, num_entries=1 << 20, num_kv_heads=32, kept=None) != LONG and "null" in message()


# A cache of 8 pages of 16 tokens and 8 heads: 2^17 bytes of one-byte codes a pool, 2^18 of fp16; arrays elsewhere.
K, V, SCALES, TABLE, BEGIN, START, SLOTS, FAR = (A + (i << 20) for i in range(8))
PLACES = dict(k_cache=K, v_cache=V, kv_scales=SCALES, block_table=TABLE, tok_begin=BEGIN, start_pos=START, slot_ids=SLOTS)
ROW = 8 * 128 * 2


@pytest.mark.parametrize("out", [K, K + (1 << 17) - 2048, K - 3 * ROW - 2048 + 16, V, V + (1 << 17) - 16, SCALES, SCALES - 16,
                                 SCALES + 8 * 8 * 2 - 16, TABLE, TABLE + 16, BEGIN, START, SLOTS - 16])
def test_outputs_in_what_the_call_reads_are_refused(out):
    """Four tokens' rows of 2048 bytes that share a byte with a pool, its scales, the table or the entries."""
    assert attend(q=rows(in_=FAR, out=out), **PLACES) == BAD and "overlaps the cache" in message(), message()
    assert read(k=out, v=FAR, **PLACES) == BAD and "overlaps the cache" in message(), message()
    assert read(k=FAR, v=out, **PLACES) == BAD and "overlaps the cache" in message(), message()


def test_only_what_a_pool_holds_is_its():
    """Wider rows for fp32; pools of fp16 are twice as long, without scales nothing is read of them."""
    end = V + (1 << 17)
    assert read(k=end - 8, v=FAR, **PLACES) == BAD and "aligned" in message()
    for at, kw in ((end - 16, dict(type=0)), (V - 3 * 4096 - 4080, dict(type=2)), (V + (1 << 18) - 16, dict(dtype=pa_amd.FP16))):
        assert read(k=at, v=FAR, **kw, **PLACES) == BAD and "overlaps the cache" in message(), message()
    assert attend(dtype=pa_amd.FP16, q=rows(in_=FAR, out=V + (1 << 18) - 16), **PLACES) == BAD and "overlaps the cache" in message()
    # A table that is said to have 2^62 entries reaches over everything behind it.
    huge = {**PLACES, "num_table_rows": 2**31 - 1, "block_table_stride": 2**31 - 1}
    assert attend(q=rows(in_=FAR, out=FAR + (1 << 19)), **huge) == BAD and "overlaps the cache" in message()
    assert attend(q=rows(in_=FAR + (1 << 19), out=FAR), tree=FAR + 4 * ROW - 8, words=1, **PLACES) == BAD and "tree" in message()
