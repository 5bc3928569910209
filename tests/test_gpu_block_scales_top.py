"""GPU tests of block-scaled caches at the largest scale that appends choose, 2^8, whose codes stop at 240."""

from __future__ import annotations

import numpy as np
import pytest

import new_tokens as nt
import pa_amd
from helpers import D, normal_f16, to_device
from test_gpu_block_scales import check_decode, dev, paged
from test_gpu_new_tokens import half, stored

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("P", [8, 16, 24])
def test_decode_at_the_largest_scale(which, P):
    """Keys (under queries so small that scores stay moderate), and values: up to 240 * 2^8 = 61440."""
    import torch
    rng = np.random.default_rng(78 + P)
    lens, hq, hkv = [100, 17, 1], 16, 4
    dk, dv, scales, table, rows = paged(rng, lens, hkv, P, hot=(which, 8))
    assert max(np.abs(r[which]).max() for r in rows) == 61440
    qb = (rng.standard_normal((3, hq, D)) * 2.0 ** (-13 if which == 0 else -5)).astype(np.float16).view(np.uint16)
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    lt = torch.tensor(lens, dtype=torch.int32)
    d.plan(lt)
    out = d.run(half(qb), dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=scales)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    check_decode(out, qb, rows)


@pytest.mark.parametrize("P", [16, 24])
def test_largest_values_appended_and_decoded(P):
    """fp16's largest values and infinities go in and come out finite: V saturates at 61440, blocks beside them keep
    their own scales."""
    import torch
    rng = np.random.default_rng(3 + P)
    n, hq, hkv = 60, 8, 2
    cols = -(-n // P)
    kb, vb = normal_f16(rng, (n, hkv, D)), normal_f16(rng, (n, hkv, D))
    v = vb.view(np.float16)
    v[20:24] = rng.choice([65504.0, -65504.0, 61440.0, 63000.0, 57344.0, 1000.0], (4, hkv, D)).astype(np.float16)
    v[22, 0, 5], v[23, 1, 7] = np.inf, -np.inf
    k_cache, v_cache = (torch.zeros((cols, hkv, P, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = pa_amd.alloc_kv_scales(cols, hkv, P)
    table = rng.permutation(cols).astype(np.int32)
    pool = nt.BlockPool(np.zeros((cols, hkv, P, D), np.uint8), scales.cpu().numpy()[..., 1])
    for lo, c in ((0, 22), (22, 38)):
        pa_amd.append_rope(None, half(kb[lo:lo + c]), half(vb[lo:lo + c]), k_cache, v_cache, to_device(table[None]),
                           dev([0, c]), dev([lo]), kv_scales=scales)
        pool.append(nt.f16(vb[lo:lo + c]), lo, table)
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    lt = torch.tensor([n], dtype=torch.int32)
    d.plan(lt)
    qb = normal_f16(rng, (1, hq, D))
    out = d.run(half(qb), k_cache, v_cache, to_device(table[None]), lt.cuda(), 1.0, 1.0, kv_scales=scales)
    torch.cuda.synchronize()
    assert np.array_equal(v_cache.cpu().numpy(), pool.codes)
    assert pool.exps.max() == 8 and pool.exps.min() < 0 and np.abs(pool.values()).max() == 61440
    assert torch.isfinite(out).all()
    rows = stored([k_cache.cpu().numpy(), v_cache.cpu().numpy()], scales.cpu().numpy(), table, n, P, 1.0)
    check_decode(out, qb, [rows])
