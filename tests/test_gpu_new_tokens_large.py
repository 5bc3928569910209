"""GPU tests of the new-token operators at sizes where their large-call kernels run (four row groups a wave from 8192
groups on, loads past the caches and another order of the grid from 96 MiB of rows on). The
reference is the definitions in 64 bits, computed by elementary operations on the device (tests/new_tokens.py has them on
the host, and the tolerances)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import new_tokens as nt
import pa_amd
from helpers import D, to_device
from test_gpu_new_tokens import DTYPES, bits, cache_view

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]

HQ, HKV = 18, 5   # five and two groups of four rows, the last ones partly filled: 7 groups a token, 9 with the values


def heads(g, n, hq=HQ, hkv=HKV):
    """q, k and v [n, heads, 128]: columns of one buffer, with NaN behind them."""
    x = torch.empty((n, hq + 2 * hkv + 1, D), dtype=torch.float16, device="cuda").normal_(generator=g)
    x[:, hq + 2 * hkv:] = float("nan")
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:hq + 2 * hkv]


def rotated(x, w, eps, pos, rot, axis, interleaved):
    """x [n, h, 128] normed and rotated in 64 bits, and |a| + |b| of each dim's pair. pos [n, axes], below 2^20: an
    angle is then off by 2^-33."""
    x = x.double()
    if w is not None:
        x = x * w.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y, mag, m = x.clone(), x.abs(), rot // 2
    if m:
        at = pos.double()[:, torch.zeros(m, dtype=torch.long, device="cuda") if axis is None else torch.from_numpy(axis).cuda()]
        angle = at * torch.from_numpy(nt.freqs(rot)).cuda()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        lo, hi = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if interleaved else (slice(0, m), slice(m, 2 * m))
        a, b = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
        mag[..., lo] = mag[..., hi] = a.abs() + b.abs()
    return y, mag


def f16_tol(ref, mag):
    return ref.abs() * 2.0 ** -11 * (1 + 2.0 ** -10) + mag * nt.F32_REL + 2.0 ** -25


def e4m3_tol(ref, mag, scale):
    return torch.maximum((ref.abs() + mag * nt.F32_REL) * 2.0 ** -4, scale * 2.0 ** -10) + mag * nt.F32_REL


def near(got, ref, tol):
    over = (got.double() - ref).abs() - tol
    assert bool((over <= 0).all()), float(over.max())


def check_rows(got, x, w, eps, pos, rot, axis, interleaved):
    for lo in range(0, x.shape[0], 4096):   # (a few hundred MB of 64-bit values at a time)
        part = slice(lo, lo + 4096)
        ref, mag = rotated(x[part], w, eps, pos[part], rot, axis, interleaved)
        near(got[part], ref, f16_tol(ref, mag))


@pytest.mark.parametrize("n", [1173, 17099], ids=["four-groups", "streamed"])
@pytest.mark.parametrize("rot,interleaved,axes,norm", [
    (128, False, 1, True), (128, True, 3, False), (96, False, 2, True), (64, True, 1, True), (0, False, 1, True)])
def test_norm_rope_large(n, rot, interleaved, axes, norm):
    g = torch.Generator(device="cuda").manual_seed(n + rot)
    q, k, v = heads(g, n)
    pos = torch.randint(0, 200000, (n, axes), device="cuda", generator=g).to(torch.int32)
    axis = None if axes == 1 else np.arange(rot // 2) % axes
    rope = pa_amd.Rope(nt.freqs(rot), axes=axis, interleaved=interleaved, num_axes=axes) if rot else None
    w = 1.0 + 0.2 * torch.empty(D, device="cuda").normal_(generator=g) if norm else None
    before = q.clone()
    qo, ko = pa_amd.norm_rope(q, k, pos, rope, q_weight=w, k_weight=w, eps=1e-5)
    eps = float(np.float32(1e-5))
    for got, x in ((qo, q), (ko, k)):
        check_rows(got, x, w, eps, pos, rot, axis, interleaved)
    assert torch.equal(q, before)


def layout(rng, n, P, entries, far):
    """Ragged entries of n tokens at ragged places (among them an empty one), and their pages in any order:
    (tok_begin, starts, table, each token's entry and place)."""
    cut = np.sort(rng.integers(0, n + 1, entries - 1))
    begin = np.concatenate([[0], cut, [n]])
    begin[2] = begin[1]
    starts = rng.integers(0, far, entries)
    counts = np.diff(begin)
    cols = int((starts + counts).max()) // P + 1
    table = rng.permutation(entries * cols + 3)[:entries * cols].reshape(entries, cols).astype(np.int32)
    e = np.repeat(np.arange(entries), counts)
    return begin.astype(np.int32), starts.astype(np.int32), table, e, starts[e] + np.arange(n) - begin[e]


def codes(x):
    """E4M3 codes of 64-bit values of at most 448, nearest ones, even ones of two (every product here is exact in 32
    bits)."""
    return x.float().to(torch.float8_e4m3fn).view(torch.uint8)


def values(c):
    return c.view(torch.float8_e4m3fn).double()


@pytest.mark.parametrize("n", [1001, 14051], ids=["four-groups", "streamed"])
@pytest.mark.parametrize("kind,P", [("fp16", 16), ("fp8", 24), ("block", 16), ("block", 24)])
@pytest.mark.parametrize("rot,interleaved", [(128, False), (128, True), (96, False)])
def test_append_rope_large(n, kind, P, rot, interleaved):
    rng = np.random.default_rng(n + P + rot)
    g = torch.Generator(device="cuda").manual_seed(n + P)
    q, k, v = heads(g, n)
    begin, starts, table, e, place = layout(rng, n, P, 7, 3 * P)
    pages = int(table.max()) + 4
    dt = torch.float16 if kind == "fp16" else torch.uint8
    shape = (pages, HKV, P, D)
    if kind == "fp16":
        pools = [torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2)]
    else:
        pools = [torch.randint(0, 0x70, shape, dtype=dt, device="cuda", generator=g) for _ in range(2)]
    scale = 0.0125 if kind == "fp8" else 1.0
    B = nt.block_tokens(P)
    scales = torch.randint(110, 124, (pages, HKV, P // B, 2), dtype=torch.uint8, device="cuda", generator=g) if kind == "block" else None
    was = [p.clone() for p in pools]
    was_scales = None if scales is None else scales.clone()
    w = 1.0 + 0.2 * torch.empty(D, device="cuda").normal_(generator=g)
    rope = pa_amd.Rope(nt.freqs(rot), interleaved=interleaved)
    qo = pa_amd.append_rope(q, k, v, *pools, to_device(table), to_device(begin), to_device(starts), rope, q_weight=w,
                            k_weight=w, eps=1e-5, k_scale=scale, v_scale=scale, kv_scales=scales)
    eps = float(np.float32(1e-5))
    pos = torch.from_numpy(place).cuda()
    check_rows(qo, q, w, eps, pos[:, None], rot, None, interleaved)
    page = torch.from_numpy(table[e, place // P].astype(np.int64)).cuda()
    slot = pos % P
    written = torch.zeros((pages, P), dtype=torch.bool, device="cuda")
    written[page, slot] = True
    kref, kmag = rotated(k, w, eps, pos[:, None], rot, None, interleaved)
    if kind != "block":
        for pool, old in zip(pools, was):
            assert torch.equal(pool.transpose(1, 2)[~written], old.transpose(1, 2)[~written])
        got_k, got_v = (p[page, :, slot] for p in pools)
        if kind == "fp16":
            assert torch.equal(got_v, v)
            near(got_k, kref, f16_tol(kref, kmag))
        else:
            inv = np.float32(1.0) / np.float32(scale)
            assert torch.equal(got_v, codes((v.float() * float(inv)).clamp(-448, 448)))
            s = float(np.float32(scale))
            kref = kref.clamp(-448 * s, 448 * s)
            near(values(got_k) * s, kref, e4m3_tol(kref, kmag, torch.tensor(s, dtype=torch.float64, device="cuda")))
        return
    # Blocks: what their tokens ask for; the first block of an entry may hold earlier rows.
    nb = P // B
    blk = page * nb + slot // B
    for j, (pool, old, x, slack) in enumerate(((pools[0], was[0], kref, nt.F32_REL), (pools[1], was[1], v.double(), 0.0))):
        lim = kmag if j == 0 else x.abs()
        big = torch.zeros((pages * nb, HKV), dtype=torch.float64, device="cuda")
        amax = x.abs().amax(-1)
        big = big.scatter_reduce(0, blk[:, None].expand(-1, HKV), amax, "amax")
        room = torch.zeros_like(big).scatter_reduce(0, blk[:, None].expand(-1, HKV), lim.amax(-1) * slack, "amax")
        need = [torch.ceil(torch.log2((big + f * room).clamp_min(1e-30) / 448.0)).clamp(-32, 8) for f in (-1, 1)]
        first = torch.full((pages * nb,), P, dtype=torch.long, device="cuda").scatter_reduce(0, blk, slot % B, "amin")
        before = was_scales[..., j].permute(0, 2, 1).reshape(pages * nb, HKV).double() - 127
        now = scales[..., j].permute(0, 2, 1).reshape(pages * nb, HKV).double() - 127
        for i, f in enumerate(need):   # (a rotated key's largest value is known to 2^-19: at a border either scale)
            need[i] = torch.where((first > 0)[:, None], torch.maximum(f, before), f)
            need[i] = torch.where((first == P)[:, None], before, need[i])
        assert bool(((now >= need[0]) & (now <= need[1])).all())
        assert int((need[0] != need[1]).sum()) <= 2 + need[0].numel() // 1000
        step = torch.exp2(now)[blk][..., None]
        got = pool[page, :, slot]
        if j == 1:
            assert torch.equal(got, codes(x / step))
        else:
            near(values(got) * step, x, e4m3_tol(x, kmag, step))
        # Every other row: as it was, or moved to its block's new scale.
        moved = torch.exp2(before - now).view(pages, nb, HKV).permute(0, 2, 1).repeat_interleave(B, dim=2)[..., None]
        earlier = torch.arange(P, device="cuda")[None] % B < first.view(pages, nb).repeat_interleave(B, dim=1)
        earlier &= (first != P).view(pages, nb).repeat_interleave(B, dim=1)
        want = torch.where(earlier[:, None, :, None] & (moved < 1), codes(values(old) * moved), old)
        keep = ~written
        assert torch.equal(pool.transpose(1, 2)[keep], want.transpose(1, 2)[keep])


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P,n", [(64, 1003), (2048, 14051)], ids=["four-groups", "96MiB"])
def test_cache_append_rope_large_in_arguments(kind, interleaved, P, n):
    """A long prompt of few pages, whose metadata goes in the kernel's arguments: the raw append's bytes (that one in
    parts where blocks do not ask for one call)."""
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k, v = heads(g, n)
    pages, scale = -(-n // P) + 2, 0.02 if kind == "fp8" else 1.0
    cache = pa_amd.PagedKVCache(pages, P, HKV, D, 2, pages, DTYPES[kind], scale, scale)
    cache.shuffle_free_pages(3)
    s = cache.admit()
    rope = pa_amd.Rope(nt.freqs(128), interleaved=interleaved)
    w = 1.0 + 0.2 * torch.empty(D, device="cuda").normal_(generator=g)
    qo = cache.append_rope([s], [n], k, v, rope, q=q, q_weight=w, k_weight=w)
    own = [torch.zeros((pages, HKV, P, D), dtype=torch.float16 if kind == "fp16" else torch.uint8, device="cuda") for _ in range(2)]
    scales = pa_amd.alloc_kv_scales(pages, HKV, P) if kind == "block" else None
    table = to_device(np.ascontiguousarray(cache.block_table(s))[None])
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    parts, size = [], n if kind == "block" else 499
    for lo in range(0, n, size):
        c = min(size, n - lo)
        parts.append(pa_amd.append_rope(q[lo:lo + c], k[lo:lo + c], v[lo:lo + c], *own, table, dev([0, c]), dev([lo]), rope,
                                        q_weight=w, k_weight=w, k_scale=scale, v_scale=scale, kv_scales=scales))
    torch.cuda.synchronize()
    assert torch.equal(qo, torch.cat(parts))
    pools, sc = cache_view(cache, kind, pages, HKV, P)
    t = np.arange(n)
    page, slot = cache.block_table(s)[t // P], t % P
    for a, b in zip(pools, own):
        b = bits(b) if kind == "fp16" else b.cpu().numpy()
        assert np.array_equal(a[page, :, slot], b[page, :, slot])
    if sc is not None:
        assert np.array_equal(sc[page, :, slot // 16], scales.cpu().numpy()[page, :, slot // 16])
    cache.close()
