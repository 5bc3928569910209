"""CPU tests of the drafted-token operators' limits, at their edges: what a call at a limit asks of a launch."""

from test_drafts import keep
from test_new_tokens import LONG, message

import pa_amd


def test_keep_rows_at_its_limit():
    """2^20 entries of 32 heads are 2^25 items: 2^32 threads in a block-scaled cache, which no launch has."""
    assert keep(num_entries=1 << 20, num_kv_heads=32) == LONG and "2^25 - 1" in message()
    for dtype in (pa_amd.FP16, pa_amd.FP8_E4M3, pa_amd.FP8_E4M3_BLOCK):
        assert keep(dtype=dtype, num_entries=1 << 20, num_kv_heads=33, page_size=8) == LONG and "2^25" in message()
    # One entry fewer passes the check, and so does the limit elsewhere (refused only for the missing pointer behind it).
    assert keep(num_entries=(1 << 20) - 1, num_kv_heads=32, kept=None) != LONG and "null" in message()
    for dtype in (pa_amd.FP16, pa_amd.FP8_E4M3):
        assert keep(dtype=dtype, num_entries=1 << 20, num_kv_heads=32, kept=None) != LONG and "null" in message()
