"""GPU test of outputs of the drafted-token operators right beside what the call reads: one allocation that holds pools,
scales and outputs end to end, output rows between rows of q."""

import numpy as np
import pytest
import torch

import pa_amd
from drafts import D, Cache, random_tree, tree_bits
from test_gpu_drafts import begins, check_attention, cols_for, ints

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
def test_outputs_beside_the_cache(kind):
    entries, hq = [(40, 9), (7, 20)], 4
    n = sum(m for _, m in entries)
    cache = Cache(kind, 16, 2, 2, cols_for(entries, 16), seed=3)
    k, v, table, scales = cache.device()
    sizes = [x.numel() * x.element_size() for x in (k, v)] + [0 if scales is None else scales.numel()]
    rows = n * hq * D * 2                            # of an output
    flat = torch.zeros(sum(sizes) + 5 * rows, dtype=torch.uint8, device="cuda")
    at = 0

    def take(size, like=None):
        nonlocal at
        x = flat[at:at + size]
        at += size
        if like is None:
            return x.view(torch.float16).view(n, -1, D)
        x.copy_(like.reshape(-1).view(torch.uint8))
        return x.view(like.dtype).view(like.shape)
    out0, k, out1, v, both, last = take(rows), take(sizes[0], k), take(rows), take(sizes[1], v), take(2 * rows), take(rows)
    scales = None if scales is None else take(sizes[2], scales)
    assert at == flat.numel()
    q, out2 = both[:, :hq], both[:, hq:]             # columns of one buffer
    q.copy_(torch.randn((n, hq, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    trees = [random_tree(np.random.default_rng(i), m) for i, (_, m) in enumerate(entries)]
    bits = tree_bits([x for t in trees for x in t], 1)
    starts, tb = ints(s for s, _ in entries), begins([m for _, m in entries])
    for out in (out0, out1, out2, last):
        got = pa_amd.tree_attention(q, k, v, table, tb, starts, bits, out=out, **cache.kw(scales))
        check_attention(cache, entries, hq, trees, got, q.cpu().numpy())
    for i, (k_out, v_out) in enumerate(((out0, out1), (out2, last))):
        got = pa_amd.read_cache(k, v, table, tb, starts, n, k_out=k_out[:, :2], v_out=v_out[:, 2:], **cache.kw(scales))
        for j in range(2):
            want = np.concatenate([cache.rows(j, e, s, s + m) for e, (s, m) in enumerate(entries)])
            x = got[j].double().cpu().numpy()
            assert (np.abs(x - want) <= np.abs(want) * 2.0 ** -10 + 2.0 ** -24).all(), (i, j)
    for x in (k, v):
        rows_ = x.view(-1).view(torch.float16)[:n * hq * D].view(n, hq, D)
        with pytest.raises(Exception, match="overlaps the cache"):
            pa_amd.tree_attention(q, k, v, table, tb, starts, bits, out=rows_, **cache.kw(scales))
        with pytest.raises(Exception, match="overlaps the cache"):
            pa_amd.read_cache(k, v, table, tb, starts, n, v_out=rows_[:, :2], **cache.kw(scales))
