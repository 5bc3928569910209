"""GPU tests of uses of the new-token operators that their documentation allows: operands that repeat or are one tensor,
batches without a token to store, two calls at once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import new_tokens as nt
import pa_amd
from helpers import D, normal_f16, to_device
from test_gpu_block_scales import check_decode
from test_gpu_new_tokens import CACHES, Paged, bits, check_rows, half, make_heads, stored

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def dev(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def test_one_row_turned_to_many_positions():
    """A token stride of 0: the same heads at every position."""
    rng = np.random.default_rng(1)
    b = normal_f16(rng, (1, 5, D))
    x = half(b).expand(40, 5, D)
    pos = torch.arange(40, dtype=torch.int32, device="cuda") * 977
    rope = pa_amd.Rope(nt.freqs(128))
    out, same = pa_amd.norm_rope(x, x, pos, rope)
    assert torch.equal(out, same)
    check_rows(bits(out), *nt.norm_rotate(nt.f16(np.repeat(b, 40, 0)), None, 0, pos.cpu().numpy(), nt.freqs(128)))


@pytest.mark.parametrize("kind", CACHES)
def test_keys_and_values_of_one_tensor(kind):
    rng = np.random.default_rng(2)
    P, hkv = 16, 3
    cache = Paged(rng, kind, 4, hkv, P)
    cache.begin()
    (x,), (b,) = make_heads(rng, 21, (hkv,), False)
    table = np.array([[2, 0, 3]], np.int32)
    pa_amd.append_rope(None, x, x, *cache.dev, to_device(table), dev([0, 21]), dev([7]), **cache.args())
    cache.append(nt.f16(b), np.abs(nt.f16(b)), b, 7, table[0])
    cache.check()


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("n", [5, 2000])
def test_nothing_to_store(kind, n):
    """Every entry empty: q is turned (to the given positions), the cache stays as it is."""
    rng = np.random.default_rng(3)
    P, hq, hkv = 24 if kind == "block" else 5, 6, 3
    cache = Paged(rng, kind, 4, hkv, P)
    before = [t.clone() for t in cache.dev] + ([cache.scales.clone()] if kind == "block" else [])
    (q, k, v), (qb, _, _) = make_heads(rng, n, (hq, hkv, hkv), True)
    pos = rng.integers(0, 5000, n)
    for begin in ([0, 0, 0], [n, n, n], [2, 2, 2]):
        out = pa_amd.append_rope(q, k, v, *cache.dev, dev([[0, 1], [2, 3]]), dev(begin), dev([0, 3]),
                                 pa_amd.Rope(nt.freqs(64)), positions=dev(pos), **cache.args())
        check_rows(bits(out), *nt.norm_rotate(nt.f16(qb), None, 0, pos, nt.freqs(64)))
    for a, b in zip(before, [*cache.dev] + ([cache.scales] if kind == "block" else [])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kind", CACHES)
def test_two_calls_at_once(kind):
    """Appends of different sequences of one cache, and a decode of a third one, on three streams: what they store and
    give one after the other. (Sequences lie in pages of their own; their scales share words.)"""
    rng = np.random.default_rng(4)
    P, hq, hkv, n = 16, 8, 1, 600
    cols = -(-(n + 9) // P)
    pages = 3 * cols
    table = np.arange(pages, dtype=np.int32).reshape(cols, 3).T.copy()   # pages of the three in turn
    dt = to_device(table)
    rope = pa_amd.Rope(nt.freqs(128))
    fp16 = kind == "fp16"

    def fresh():
        pools = [torch.zeros((pages, hkv, P, D), dtype=torch.float16 if fp16 else torch.uint8, device="cuda") for _ in range(2)]
        return pools + [pa_amd.alloc_kv_scales(pages, hkv, P) if kind == "block" else None]

    def append(c, row, x, start):
        return pa_amd.append_rope(x[0], x[1], x[2], c[0], c[1], dt, dev([0, x[1].shape[0]]), dev([start]), rope, kv_scales=c[2],
                                  slot_ids=dev([row]), k_scale=0.02 if kind == "fp8" else 1.0, v_scale=0.02 if kind == "fp8" else 1.0)

    parts = [[make_heads(rng, m, (hq, hkv, hkv), True)[0] for m in (9, n)] for _ in range(3)]
    want, got = fresh(), fresh()
    lens = torch.tensor([9], dtype=torch.int32)
    d = pa_amd.Decoder(hq, hkv, D, P, not fp16, **(dict(block_scales=True) if kind == "block" else {}))
    d.plan(lens)
    lens_dev, scale = lens.cuda(), 0.02 if kind == "fp8" else 1.0
    more = lambda c: dict(kv_scales=c[2]) if kind == "block" else {}   # noqa: E731
    for c in (want, got):
        for row in range(3):
            append(c, row, parts[row][0], 0)
    qd = half(normal_f16(rng, (1, hq, D)))
    ref = [append(want, row, parts[row][1], 9) for row in range(2)]
    ref.append(d.run(qd, want[0], want[1], dt[2:].contiguous(), lens_dev, scale, scale, **more(want)))
    last = dt[2:].contiguous()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for row, s in enumerate(streams):
        with torch.cuda.stream(s):
            if row < 2:
                outs.append(append(got, row, parts[row][1], 9))
            else:
                outs.append(d.run(qd, got[0], got[1], last, lens_dev, scale, scale, **more(got)))
    torch.cuda.synchronize()
    for a, b in zip(ref, outs):
        assert torch.equal(a, b)
    for a, b in zip(want, got):
        assert a is None or torch.equal(a, b)
    pools = [bits(t) if fp16 else t.cpu().numpy() for t in got[:2]]
    rows = stored(pools, None if got[2] is None else got[2].cpu().numpy(), table[2], 9, P, scale)
    check_decode(outs[2], bits(qd), [rows])
