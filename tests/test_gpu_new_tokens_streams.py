"""GPU tests of appends that are given a stream other than the current one."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import new_tokens as nt
import pa_amd
from helpers import D
from test_gpu_new_tokens import DTYPES, CACHES, bits, make_heads

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def stream_of(t) -> int:
    """The stream that torch's allocator keeps this tensor's memory for."""
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= t.data_ptr() < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not torch's memory")


@pytest.mark.parametrize("kind", CACHES)
def test_new_output_belongs_to_the_given_stream(kind):
    """The output that append_rope makes is the given stream's memory (whatever way the stream is given), not a block
    that work queued on the current stream may still use; where none is given, the current one's."""
    rng = np.random.default_rng(1)
    cache = pa_amd.PagedKVCache(8, 16, 2, D, 2, 4, DTYPES[kind])
    s = cache.admit()
    rope = pa_amd.Rope(nt.freqs(128))
    (q, k, v), _ = make_heads(rng, 3, (8, 2, 2), True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    current = torch.cuda.current_stream().cuda_stream
    at = 0
    for stream, owner in ((side, side.cuda_stream), (side.cuda_stream, side.cuda_stream), (None, current),
                          (torch.cuda.current_stream(), current)):
        spare = torch.empty((3, 8, D), dtype=torch.float16, device="cuda")
        del spare   # a block of the output's size, free on the current stream
        out = cache.append_rope([s], [3], k, v, rope, q=q, stream=stream)
        torch.cuda.synchronize()
        assert stream_of(out) == owner
        place = torch.arange(at, at + 3, dtype=torch.int32, device="cuda")
        assert np.array_equal(bits(out), bits(pa_amd.norm_rope(q, None, place, rope)[0]))
        at += 3
    with torch.cuda.stream(side):   # the current one's handle given while another is current
        out = cache.append_rope([s], [3], k, v, rope, q=q, stream=torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    assert stream_of(out) == torch.cuda.default_stream().cuda_stream
    cache.close()
