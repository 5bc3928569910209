"""GPU tests of what the paged cache's appends refuse of their operands (a cache needs a device): nothing is launched and
nothing changes."""

from __future__ import annotations

import pytest
import torch

import pa_amd
from helpers import D
from test_gpu_new_tokens import CACHES, DTYPES

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


@pytest.mark.parametrize("kind", CACHES)
def test_appends_refuse_null_and_unaligned_tokens(kind):
    cache = pa_amd.PagedKVCache(4, 16, 2, D, 2, 4, DTYPES[kind])
    s = cache.admit()
    x = torch.zeros(5 * 2 * D + 8, dtype=torch.float16, device="cuda")
    good, odd = x.data_ptr(), x.data_ptr() + 2
    bad = [(None, good), (good, None)] + ([(odd, good), (good, odd), (good + 8, good)] if kind == "block" else [])
    for k, v in bad:
        for call in (lambda: cache.append(s, k, v, 5), lambda: cache.append_batch([s], [5], k, v)):
            with pytest.raises(pa_amd.InvalidArgument, match="null|aligned"):
                call()
            assert cache.seq_len(s) == 0 and cache.free_pages() == 4
    assert cache.append(s, None, None, 0) and cache.append_batch([s], [0], None, None)   # no tokens: nothing is read
    assert cache.append(s, good, good, 5) and cache.append_batch([s], [5], good, good)
    assert cache.seq_len(s) == 10
    cache.close()


@pytest.mark.parametrize("scale", [0.0, 1e-39, float("inf"), float("nan")])
def test_append_rope_refuses_a_cache_without_reciprocals(scale):
    """A per-tensor FP8 cache whose scale no value can be divided by (the raw append refuses such scales, too)."""
    x = torch.zeros((3, 2, D), dtype=torch.float16, device="cuda")
    for k_scale, v_scale in ((scale, 1.0), (1.0, scale)):
        cache = pa_amd.PagedKVCache(4, 16, 2, D, 2, 4, pa_amd.FP8_E4M3, k_scale, v_scale)
        s = cache.admit()
        with pytest.raises(pa_amd.InvalidArgument, match="reciprocals"):
            cache.append_rope([s], [3], x, x)
        assert cache.seq_len(s) == 0 and cache.free_pages() == 4
        cache.close()
