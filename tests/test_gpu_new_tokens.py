"""GPU tests of head norms with rotation and of appends with rotation, against the definitions in 64 bits (and, for what
passes as it is, bit for bit against the oracle)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import new_tokens as nt
import oracle
import pa_amd
from helpers import D, d2h, normal_f16, to_device
from pa_amd import _lib

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


@pytest.fixture(params=["compiled", "ctypes"])
def binding(request, monkeypatch):
    """Both bindings of the torch operators."""
    from pa_amd import ops
    if request.param == "ctypes":
        monkeypatch.setattr(ops, "compiled", lambda: None)
    else:
        assert ops.compiled() is not None
    return request.param


def half(a):
    import torch
    return to_device(np.asarray(a, np.uint16)).view(torch.float16)


def bits(t) -> np.ndarray:
    import torch
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def make_heads(rng, n, heads, fused):
    """Device tensors [n, h, 128] for each of `heads`, and their fp16 bits; columns of one buffer if fused."""
    import torch
    arrays = [normal_f16(rng, (n, h, D)) for h in heads]
    if not fused:
        return [half(a) for a in arrays], arrays
    buf = torch.full((n, sum(heads) + 1, D), float("nan"), dtype=torch.float16, device="cuda")
    out, at = [], 0
    for h, a in zip(heads, arrays):
        buf[:, at:at + h] = half(a)
        out.append(buf[:, at:at + h])
        at += h
    return out, arrays


def weights(rng, norm):
    import torch
    if not norm:
        return None, None
    w = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    return torch.from_numpy(w).cuda(), w


def check_rows(got, ref, mag):
    err = np.abs(nt.f16(got) - ref)
    assert np.all(err <= nt.f16_tol(ref, mag)), float((err - nt.f16_tol(ref, mag)).max())


ROT = [  # rot, interleaved, axes, norm, fused
    (128, False, 1, True, True), (128, True, 1, True, False), (64, False, 1, False, True), (96, False, 3, True, True),
    (96, True, 2, False, False), (16, False, 1, True, False), (16, True, 4, True, True), (32, False, 1, False, False),
    (0, False, 1, True, True),
]


@pytest.mark.parametrize("rot,interleaved,axes,norm,fused", ROT)
@pytest.mark.parametrize("n,hq,hkv", [(1, 32, 8), (3, 5, 1), (257, 8, 3), (66, 1, 2)])
def test_norm_rope(binding, n, hq, hkv, rot, interleaved, axes, norm, fused):
    import torch
    rng = np.random.default_rng(n * 1000 + rot)
    (q, k), (qb, kb) = make_heads(rng, n, (hq, hkv), fused)
    pos = rng.integers(0, 200000, (n, axes))
    pos[0] = [0, 1, -5, 2**31 - 1][:axes]
    pos[n // 2, 0] = 2**31 - 1
    pos[-1, -1] = -2**31
    axis = None if axes == 1 else np.arange(rot // 2) % axes
    rope = pa_amd.Rope(nt.freqs(rot), axes=axis, interleaved=interleaved, scale=1.25, num_axes=axes) if rot else None
    wq, wqf = weights(rng, norm)
    wk, wkf = weights(rng, norm)
    p = torch.from_numpy(pos.astype(np.int32)).cuda()
    qo, ko = pa_amd.norm_rope(q, k, p if axes > 1 else p[:, 0].contiguous(), rope, q_weight=wq, k_weight=wk, eps=1e-5)
    torch.cuda.synchronize()
    for got, b, w in ((qo, qb, wqf), (ko, kb, wkf)):
        fr = nt.freqs(rot) if rot else None
        ref, mag = nt.norm_rotate(nt.f16(b), w, float(np.float32(1e-5)), pos, fr, axis, interleaved, 1.25)
        assert got.shape == b.shape and got.is_contiguous()
        check_rows(bits(got), ref, mag)
    assert np.array_equal(bits(q), qb) and np.array_equal(bits(k), kb)   # inputs stay


@pytest.mark.parametrize("rot,interleaved", [(128, False), (128, True), (96, False)])
def test_norm_rope_in_place_and_alone(rot, interleaved):
    """q in place in a fused buffer, k None, and the other way round: equal to the call with new outputs, bit for bit."""
    import torch
    rng = np.random.default_rng(3)
    rope = pa_amd.Rope(nt.freqs(rot), interleaved=interleaved)
    wq, _ = weights(rng, True)
    pos = torch.arange(37, dtype=torch.int32, device="cuda") * 1000
    (q, k, v), (_, kb, vb) = make_heads(rng, 37, (8, 2, 2), True)
    want_q, want_k = pa_amd.norm_rope(q, k, pos, rope, q_weight=wq)
    a, none = pa_amd.norm_rope(q, None, pos, rope, q_weight=wq, q_out=q)
    assert none is None and a.data_ptr() == q.data_ptr()
    assert np.array_equal(bits(q), bits(want_q)) and np.array_equal(bits(k), kb) and np.array_equal(bits(v), vb)
    none, b = pa_amd.norm_rope(None, k, pos, rope, k_out=k)
    assert none is None and np.array_equal(bits(b), bits(want_k)) and np.array_equal(bits(v), vb)


def test_norm_rope_special_values():
    """Zero rows, infinities, NaN and the largest values: a row's own, none of its neighbours'; dims past the rotation
    and rows without a norm keep theirs."""
    import torch
    n = 6
    x = np.ones((n, 3, D), np.float16)
    x[0] = 0
    x[1, 1, 3], x[2, 0, 100], x[3, 2, 127] = np.inf, np.nan, -np.inf
    x[4] = 65504
    x[5] = 6e-8
    q = half(x.view(np.uint16))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    w = torch.ones(D, device="cuda")
    rope = pa_amd.Rope(nt.freqs(64))
    plain, _ = pa_amd.norm_rope(q, None, pos, rope)
    normed, _ = pa_amd.norm_rope(q, None, pos, rope, q_weight=w)
    p, m = plain.float().cpu().numpy(), normed.float().cpu().numpy()
    xf = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        ref, _ = nt.norm_rotate(xf, None, 0, np.arange(n), nt.freqs(64))
        refn, _ = nt.norm_rotate(xf, np.ones(D), float(np.float32(1e-6)), np.arange(n), nt.freqs(64))
    for got, want in ((p, ref), (m, refn)):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        big = np.abs(want) >= 65520   # rounds to infinity
        assert np.array_equal(np.isinf(got), big)
        ok = np.isfinite(want) & ~big
        assert np.all(np.abs(got[ok] - want[ok]) <= np.abs(want)[ok] * 2.0 ** -10 + 2.0 ** -17)
    assert np.all(m[0] == 0) and np.isinf(p[3, 2, 127]) and np.isfinite(p[3, 2, :127]).all()


def test_norm_rope_refuses(binding):
    import torch
    q = torch.zeros((4, 2, D), dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    rope = pa_amd.Rope(nt.freqs(128))
    two = pa_amd.Rope(nt.freqs(128), axes=np.arange(64) % 2)
    w = torch.ones(D, device="cuda")
    bad = [
        dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :, :64]), dict(q=q.transpose(0, 1)), dict(q=q[0]),
        dict(k=torch.zeros((5, 2, D), dtype=torch.float16, device="cuda")), dict(q=None, k=None),
        dict(positions=None), dict(positions=pos.long()), dict(positions=pos[:3]), dict(positions=pos.cpu()),
        dict(rope=two), dict(q_weight=w.half()), dict(q_weight=w[:64]), dict(q_weight=w.cpu()),
        dict(q_out=torch.empty_like(q)[:3]), dict(q_out=torch.empty((4, 3, D), dtype=torch.float16, device="cuda")),
        dict(eps=-1.0, q_weight=w), dict(q=torch.zeros((4 * 2 * D + 4,), dtype=torch.float16, device="cuda")[4:].view(4, 2, D)),
    ]
    for change in bad:
        args = dict(q=q, k=None, positions=pos, rope=rope) | change
        qq, kk, pp, rr = (args.pop(x) for x in ("q", "k", "positions", "rope"))
        with pytest.raises((RuntimeError, ValueError)):
            pa_amd.norm_rope(qq, kk, pp, rr, **args)
    # An output that overlaps the rows other than as themselves.
    buf = torch.zeros((5, 2, D), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        pa_amd.norm_rope(buf[:4], None, pos, rope, q_out=buf[1:])
    out, _ = pa_amd.norm_rope(torch.empty((0, 2, D), dtype=torch.float16, device="cuda"), None, pos[:0], rope)
    assert out.shape == (0, 2, D)


CACHES = ["fp16", "fp8", "block"]


class Paged:
    """A caller's cache and a plain copy of it, for raw appends."""

    def __init__(self, rng, kind, pages, hkv, P):
        import torch
        self.kind, self.P, self.hkv, self.pages = kind, P, hkv, pages
        shape = (pages, hkv, P, D)
        if kind == "fp16":
            self.host = [rng.integers(0, 0x7C00, shape, dtype=np.uint16) for _ in range(2)]
            self.dev = [half(a) for a in self.host]
        else:
            self.host = [rng.integers(0, 0x7F, shape, dtype=np.uint8) for _ in range(2)]
            self.dev = [to_device(a) for a in self.host]
        self.scale = (0.0125, 0.011) if kind == "fp8" else (1.0, 1.0)
        self.scales, self.pools = None, None
        if kind == "block":
            b = nt.block_tokens(P)
            sc = rng.integers(110, 130, (pages, hkv, P // b, 2), dtype=np.uint8)
            self.scales = torch.from_numpy(sc).cuda()
            self.pools = [nt.BlockPool(self.host[j], sc[..., j]) for j in range(2)]

    def args(self):
        return dict(k_scale=self.scale[0], v_scale=self.scale[1], kv_scales=self.scales)

    def append(self, k, mag, vb, start, table):
        """Plain: k [n, hkv, 128] float64 (what it is computed from: mag), v fp16 bits."""
        for i in range(k.shape[0]):
            page, slot = table[(start + i) // self.P], (start + i) % self.P
            if self.kind == "fp16":
                self.host[1][page, :, slot] = vb[i]
            elif self.kind == "fp8":
                inv = np.float32(1.0) / np.float32(self.scale[1])
                self.host[1][page, :, slot] = oracle.f32_to_e4m3(
                    (vb[i].view(np.float16).astype(np.float32) * inv)).reshape(self.hkv, D)
            self.written[page, :, slot] = True
            self.k_ref[page, :, slot], self.k_mag[page, :, slot] = k[i], mag[i]
        if self.kind == "block":
            self.pools[0].append(k, start, table)
            self.pools[1].append(nt.f16(vb), start, table)

    def begin(self):
        shape = (self.pages, self.hkv, self.P, D)
        self.written = np.zeros(shape[:3], bool)
        self.k_ref, self.k_mag = np.zeros(shape), np.zeros(shape)

    def check(self):
        """The device's pools: v bit for bit, k within its type's half step, everything else as it was (block-scaled:
        what an earlier row of a grown block becomes is the plain pool's)."""
        import torch
        torch.cuda.synchronize()
        if self.kind == "fp16":
            k, v = (bits(t) for t in self.dev)
            assert np.array_equal(v, self.host[1])
            assert np.array_equal(k[~self.written], self.host[0][~self.written])
            err = np.abs(nt.f16(k) - self.k_ref)[self.written]
            assert np.all(err <= nt.f16_tol(self.k_ref, self.k_mag)[self.written])
            return
        k, v = (t.cpu().numpy() for t in self.dev)
        if self.kind == "fp8":
            assert np.array_equal(v, self.host[1])
            assert np.array_equal(k[~self.written], self.host[0][~self.written])
            s = float(np.float32(self.scale[0]))
            ref = np.clip(self.k_ref, -448 * s, 448 * s)
            err = np.abs(nt.e4m3(k) * s - ref)[self.written]
            assert np.all(err <= nt.e4m3_tol(ref, self.k_mag, s)[self.written])
            return
        sc = self.scales.cpu().numpy().astype(int) - 127
        b = nt.block_tokens(self.P)
        assert np.array_equal(sc[..., 1], self.pools[1].exps)
        assert np.array_equal(v, self.pools[1].codes)
        # k's largest value is exact to 2^-19: its scale may be the other one only where it lies that near a border.
        same = sc[..., 0] == self.pools[0].exps
        assert same.all(), np.argwhere(~same)[:5]
        step = np.repeat(2.0 ** sc[..., 0], b, axis=2)[..., None]
        err = np.abs(nt.e4m3(k) * step - self.k_ref)[self.written]
        # A row that its block's growth rounded again is off by half a step of the coarser grid more.
        assert np.all(err <= (nt.e4m3_tol(self.k_ref, self.k_mag, step) + step * 2.0 ** -10)[self.written])
        assert np.array_equal(k[~self.written], self.pools[0].codes[~self.written])


@pytest.mark.parametrize("kind,P", [("fp16", 16), ("fp16", 5), ("fp8", 16), ("fp8", 1), ("fp8", 100), ("block", 8),
                                    ("block", 16), ("block", 24), ("block", 48), ("block", 64)])
@pytest.mark.parametrize("rot,interleaved,norm,hq,hkv,fused,with_pos", [
    (128, False, True, 32, 8, True, False), (64, True, False, 0, 1, False, True), (96, False, True, 6, 3, True, True),
    (0, False, False, 4, 12, False, False)])
def test_append_rope(binding, kind, P, rot, interleaved, norm, hq, hkv, fused, with_pos):
    """Ragged entries (an empty one, one token, several pages) at ragged places, two calls one after the other, pages
    and table rows out of order."""
    import torch
    rng = np.random.default_rng(P * 10 + rot)
    counts, starts = [3, 0, 1, 2 * P + 5, 17], [P, 4, 2 * P - 1, 3, 0]
    rows = [4, 0, 2, 5, 1]
    cols = max(-(-(s + n + 9) // P) for s, n in zip(starts, counts)) + 1
    pages = 6 * cols + 1
    table = rng.permutation(pages)[:6 * cols].reshape(6, cols).astype(np.int32)
    cache = Paged(rng, kind, pages, hkv, P)
    cache.begin()
    fr = nt.freqs(rot) if rot else None
    rope = pa_amd.Rope(fr, interleaved=interleaved) if rot else None
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    for _ in range(2):
        n = sum(counts)
        heads = ([hq] if hq else []) + [hkv, hkv]
        t, b = make_heads(rng, n, heads, fused)
        q, qb = (t[0], b[0]) if hq else (None, None)
        (k, v), (kb, vb) = t[-2:], b[-2:]
        wk, wkf = weights(rng, norm)
        place = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)])
        pos = rng.integers(0, 100000, n) if with_pos else place
        qo = pa_amd.append_rope(q, k, v, *cache.dev, to_device(table), dev(np.concatenate([[0], np.cumsum(counts)])),
                                dev(starts), rope, positions=dev(pos) if with_pos else None, q_weight=wk, k_weight=wk,
                                eps=1e-5, slot_ids=dev(rows), **cache.args())
        ref, mag = nt.norm_rotate(nt.f16(kb), wkf, float(np.float32(1e-5)), pos, fr, None, interleaved)
        at = 0
        for r, s, c in zip(rows, starts, counts):
            cache.append(ref[at:at + c], mag[at:at + c], vb[at:at + c], s, table[r])
            at += c
        cache.check()
        assert (qo is None) == (not hq)
        if hq:
            ref, mag = nt.norm_rotate(nt.f16(qb), wkf, float(np.float32(1e-5)), pos, fr, None, interleaved)
            check_rows(bits(qo), ref, mag)
        starts = [s + c for s, c in zip(starts, counts)]
        counts = [1, 2, 0, 1, 9]


@pytest.mark.parametrize("kind", CACHES)
def test_append_rope_leaves_out_what_is_out_of_range(kind):
    """Places before 0 and past the table, rows and pages that do not exist: those tokens are left out, the others and
    every q row are not."""
    import torch
    rng = np.random.default_rng(8)
    P, hkv, hq, pages = 16, 2, 4, 6
    cache = Paged(rng, kind, pages, hkv, P)
    cache.begin()
    table = np.array([[0, 1], [2, 99], [-3, 3], [4, 5], [5, 4]], np.int32)
    #        fine    past page 99  page -3   row 7   row -1  past the table  before 0     at 2^31
    starts = [14,     12,          8,        0,      0,      30,             -5,          2**31 - 2]
    rows = [0,        1,           2,        7,      -1,     3,              4,           4]
    counts = [4,      8,           10,       3,      3,      6,              3,           4]
    n = sum(counts)
    (q, k, v), (qb, kb, vb) = make_heads(rng, n, (hq, hkv, hkv), False)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    qo = pa_amd.append_rope(q, k, v, *cache.dev, to_device(table), dev(np.concatenate([[0], np.cumsum(counts)])),
                            dev(starts), None, slot_ids=dev(rows), **cache.args())
    at = np.concatenate([[0], np.cumsum(counts)])
    for e, (lo, hi) in enumerate([(0, 4), (0, 4), (8, 10), (0, 0), (0, 0), (0, 2)]):
        if hi > lo:
            part = slice(at[e] + lo, at[e] + hi)
            cache.append(nt.f16(kb[part]), np.abs(nt.f16(kb[part])), vb[part], starts[e] + lo, table[rows[e]])
    cache.check()
    assert np.array_equal(bits(qo), qb)


@pytest.mark.parametrize("kind", CACHES)
def test_append_rope_replayed(kind):
    """A captured append follows the device arrays from replay to replay, beside eager work."""
    import torch
    rng = np.random.default_rng(9)
    P, hkv, hq, pages, m = 16, 2, 8, 12, 3
    cache = Paged(rng, kind, pages, hkv, P)
    rope = pa_amd.Rope(nt.freqs(128))
    table = np.arange(12, dtype=np.int32).reshape(3, 4)[:, ::-1].copy()
    (q, k, v), _ = make_heads(rng, m, (hq, hkv, hkv), False)
    starts = torch.tensor([0, 15, 31], dtype=torch.int32, device="cuda")
    begin = torch.arange(m + 1, dtype=torch.int32, device="cuda")
    dt, out = to_device(table), torch.empty_like(q)
    wk, wkf = weights(rng, True)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        pa_amd.append_rope(q, k, v, *cache.dev, dt, begin, starts, rope, q_weight=wk, k_weight=wk, q_out=out, **cache.args())
    cache.begin()
    for step in range(4):
        (q2, k2, v2), (qb, kb, vb) = make_heads(rng, m, (hq, hkv, hkv), False)
        q.copy_(q2), k.copy_(k2), v.copy_(v2)
        graph.replay()
        torch.cuda.synchronize()
        place = starts.cpu().numpy()
        ref, mag = nt.norm_rotate(nt.f16(kb), wkf, float(np.float32(1e-6)), place, nt.freqs(128))
        for e in range(m):
            cache.append(ref[e:e + 1], mag[e:e + 1], vb[e:e + 1], int(place[e]), table[e])
        cache.check()
        check_rows(bits(out), *nt.norm_rotate(nt.f16(qb), wkf, float(np.float32(1e-6)), place, nt.freqs(128)))
        starts += 1


def test_append_rope_refuses(binding):
    import torch
    n, hkv, P, pages = 4, 2, 16, 3
    z = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device="cuda")   # noqa: E731
    base = dict(q=None, k=z(n, hkv, D), v=z(n, hkv, D), k_cache=z(pages, hkv, P, D, dt=torch.uint8),
                v_cache=z(pages, hkv, P, D, dt=torch.uint8), block_table=z(1, 3, dt=torch.int32),
                tok_begin=torch.tensor([0, n], dtype=torch.int32, device="cuda"), start_pos=z(1, dt=torch.int32))
    kw = dict(kv_scales=pa_amd.alloc_kv_scales(pages, hkv, P))
    pa_amd.append_rope(*base.values(), **kw)
    bad = [dict(k=z(n, 3, D)), dict(v=z(n, 3, D)), dict(v=z(n + 1, hkv, D)), dict(q=z(n + 1, 4, D)), dict(k=z(n, hkv, D).float()),
           dict(k_cache=z(pages, hkv, P, D)), dict(k_cache=z(pages, hkv, 2 * P, D, dt=torch.uint8)),
           dict(k_cache=z(pages, 4, P, D, dt=torch.uint8)), dict(block_table=z(3, dt=torch.int32)),
           dict(block_table=z(1, 3, dt=torch.int64)), dict(tok_begin=z(3, dt=torch.int32)), dict(start_pos=z(1, dt=torch.int64)),
           dict(start_pos=z(1, 1, dt=torch.int32)), dict(kv_scales=pa_amd.alloc_kv_scales(pages + 1, hkv, P)),
           dict(kv_scales=z(pages, hkv, 2, dt=torch.uint8)), dict(slot_ids=z(2, dt=torch.int32)),
           dict(positions=z(n + 1, dt=torch.int32)), dict(tok_begin=z(2, dt=torch.int32).cpu())]
    for change in bad:
        args, more = dict(base), dict(kw)
        for name, x in change.items():
            (args if name in args else more)[name] = x
        with pytest.raises((RuntimeError, ValueError)):
            pa_amd.append_rope(*args.values(), **more)
    fp16 = dict(base, k_cache=z(pages, hkv, P, D), v_cache=z(pages, hkv, P, D))
    with pytest.raises(RuntimeError, match="kv_scales"):
        pa_amd.append_rope(*fp16.values(), **kw)
    odd = dict(base, k_cache=z(pages, hkv, 12, D, dt=torch.uint8), v_cache=z(pages, hkv, 12, D, dt=torch.uint8))
    with pytest.raises(RuntimeError, match="multiple of 8"):
        pa_amd.append_rope(*odd.values(), **kw)


# ---- the paged cache's own append ------------------------------------------

DTYPES = {"fp16": pa_amd.FP16, "fp8": pa_amd.FP8_E4M3, "block": pa_amd.FP8_E4M3_BLOCK}


def cache_view(cache, kind, pages, hkv, P):
    """The cache's pools and scale exponents on the host."""
    p = cache.params()
    nbytes = pages * hkv * P * D * (2 if kind == "fp16" else 1)
    dt = np.uint16 if kind == "fp16" else np.uint8
    pools = [d2h(a, nbytes, dt).reshape(pages, hkv, P, D) for a in (p.k_cache, p.v_cache)]
    if kind != "block":
        assert not p.kv_scales
        return pools, None
    b = nt.block_tokens(P)
    return pools, d2h(p.kv_scales, pages * hkv * (P // b) * 2).reshape(pages, hkv, P // b, 2)


def stored(pools, scales, table, n, P, scale):
    """Values [n, hkv, 128] of k and v of a sequence."""
    out = []
    for j, pool in enumerate(pools):
        val = nt.f16(pool) if pool.dtype == np.uint16 else nt.e4m3(pool) * scale
        if scales is not None:
            val = val * np.repeat(2.0 ** (scales[..., j].astype(int) - 127), nt.block_tokens(P), axis=2)[..., None]
        t = np.arange(n)
        out.append(val[np.asarray(table)[t // P], :, t % P])
    return out


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("P,big", [(16, False), (24, False), (8, True)])
def test_cache_append_rope_is_the_raw_append(kind, P, big):
    """PagedKVCache.append_rope over several calls (a slot twice in one batch, empty entries, appends past the kernel
    arguments' size) stores what raw appends of the same tokens store, bit for bit; q comes out the same."""
    import torch
    rng = np.random.default_rng(P)
    hq, hkv, slots, cols = 8, 2, 4, 200 if big else 30
    pages, scale = slots * cols, 0.02 if kind == "fp8" else 1.0
    cache = pa_amd.PagedKVCache(pages, P, hkv, D, slots, cols, DTYPES[kind], scale, scale)
    cache.shuffle_free_pages(5)
    assert [cache.admit() for _ in range(slots)] == list(range(slots))
    rope = pa_amd.Rope(nt.freqs(128))
    wq, _ = weights(rng, True)
    shape = (pages, hkv, P, D)
    own = [torch.zeros(shape, dtype=torch.float16 if kind == "fp16" else torch.uint8, device="cuda") for _ in range(2)]
    scales = pa_amd.alloc_kv_scales(pages, hkv, P) if kind == "block" else None
    rounds = [([0, 1, 2, 3], [1, 37, 0, 5]), ([3, 3, 0, 3], [2, 40, 1, 3]), ([2], [1]), ([1, 2, 0, 3], [1, 1, 1, 1])]
    if big:
        rounds.insert(1, ([0, 1, 2], [P * 150, P * 149 + 3, P * 120]))
    at = [0] * slots
    for sl, counts in rounds:
        n = sum(counts)
        (q, k, v), _ = make_heads(rng, n, (hq, hkv, hkv), True)
        qo = cache.append_rope(sl, counts, k, v, rope, q=q, q_weight=wq, k_weight=wq)
        table = np.zeros((slots, cols), np.int32)
        for s in range(slots):
            t = cache.block_table(s)
            table[s, :len(t)] = t
        lo, parts = 0, []
        for s, c in zip(sl, counts):   # one raw call per entry: the same tokens, the same places
            if c:
                parts.append(pa_amd.append_rope(
                    q[lo:lo + c], k[lo:lo + c], v[lo:lo + c], *own, to_device(table),
                    torch.tensor([0, c], dtype=torch.int32, device="cuda"),
                    torch.tensor([at[s]], dtype=torch.int32, device="cuda"), rope, q_weight=wq, k_weight=wq,
                    k_scale=scale, v_scale=scale, kv_scales=scales,
                    slot_ids=torch.tensor([s], dtype=torch.int32, device="cuda")))
            lo, at[s] = lo + c, at[s] + c
        torch.cuda.synchronize()
        assert np.array_equal(bits(qo), bits(torch.cat(parts)))
        assert [cache.seq_len(s) for s in range(slots)] == at
    pools, sc = cache_view(cache, kind, pages, hkv, P)
    mine = [bits(t) if kind == "fp16" else t.cpu().numpy() for t in own]
    for s in range(slots):
        t = np.arange(at[s])
        page, slot = cache.block_table(s)[t // P], t % P
        for a, b in zip(pools, mine):
            assert np.array_equal(a[page, :, slot], b[page, :, slot])
        if sc is not None:
            b = nt.block_tokens(P)
            assert np.array_equal(sc[page, :, slot // b], scales.cpu().numpy()[page, :, slot // b])
    cache.close()


@pytest.mark.parametrize("kind", CACHES)
def test_cache_append_rope_plain_is_append_batch(kind):
    """Without rope, weights and q: the tokens that append and append_batch store, bit for bit, in the same order."""
    import torch
    rng = np.random.default_rng(12)
    hkv, P, slots, cols = 3, 16, 3, 8
    caches = [pa_amd.PagedKVCache(slots * cols, P, hkv, D, slots, cols, DTYPES[kind], *([0.02] * 2 if kind == "fp8" else [1.0] * 2))
              for _ in range(3)]
    for c in caches:
        for _ in range(slots):
            c.admit()
    for sl, counts in [([0, 1, 2], [20, 1, 33]), ([2, 0, 2], [1, 9, 2]), ([1, 0], [1, 1])]:
        n = sum(counts)
        (k, v), _ = make_heads(rng, n, (hkv, hkv), False)
        assert caches[0].append_rope(sl, counts, k, v) is True
        assert caches[1].append_batch(sl, counts, k, v)
        lo = 0
        for s, c in zip(sl, counts):
            assert caches[2].append(s, k[lo:lo + c], v[lo:lo + c], c)
            lo += c
    torch.cuda.synchronize()
    views = [cache_view(c, kind, slots * cols, hkv, P) for c in caches]
    for s in range(slots):
        n = caches[0].seq_len(s)
        vals = [stored(*v, c.block_table(s), n, P, 1.0) for v, c in zip(views, caches)]
        for j in range(2):
            assert np.array_equal(vals[0][j], vals[1][j]) and np.array_equal(vals[0][j], vals[2][j])
    for c in caches:
        c.close()


def test_cache_append_rope_refuses():
    import torch
    cache = pa_amd.PagedKVCache(2, 16, 2, D, 2, 2, pa_amd.FP8_E4M3_BLOCK)
    cache.admit()
    z = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")   # noqa: E731
    two = pa_amd.Rope(nt.freqs(128), axes=np.arange(64) % 2)
    bad = [([0], [4], z(4, 3, D), z(4, 3, D), {}), ([1], [4], z(4, 2, D), z(4, 2, D), {}),
           ([0], [4], z(5, 2, D), z(5, 2, D), {}), ([0], [4], z(4, 2, D), z(4, 2, D), dict(q=z(3, 2, D))),
           ([0], [4], z(4, 2, D), z(4, 2, D), dict(rope=two)), ([0], [-1], z(0, 2, D), z(0, 2, D), {}),
           ([0], [33], z(33, 2, D), z(33, 2, D), {})]
    for sl, c, k, v, kw in bad:
        with pytest.raises((RuntimeError, ValueError)):
            cache.append_rope(sl, c, k, v, **kw)
        assert cache.seq_len(0) == 0 and cache.free_pages() == 2
    cache.admit()
    assert cache.append_rope([0], [17], z(17, 2, D), z(17, 2, D)) is True
    assert cache.append_rope([1], [1], z(1, 2, D), z(1, 2, D)) is False   # out of pages
    assert cache.seq_len(1) == 0
    cache.close()


@pytest.mark.parametrize("kind", CACHES)
def test_cache_append_rope_captured(kind):
    """Captured, every replay stores the tokens then in k, v and q at the places of the capture."""
    import torch
    rng = np.random.default_rng(15)
    P, hq, hkv = 16, 4, 2
    cache = pa_amd.PagedKVCache(12, P, hkv, D, 2, 6, DTYPES[kind], *([0.02] * 2 if kind == "fp8" else [1.0] * 2))
    for _ in range(2):
        cache.admit()
    rope = pa_amd.Rope(nt.freqs(64), interleaved=True)
    (k0, v0), (kb0, vb0) = make_heads(rng, 20, (hkv, hkv), False)
    k0, v0 = k0 * 0.25, v0 * 0.25
    assert cache.append_rope([0], [20], k0, v0, rope)
    (q, k, v), _ = make_heads(rng, 2, (hq, hkv, hkv), False)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert cache.append_rope([0, 1], [1, 1], k, v, rope, q=q, q_out=out) is out
    eager = pa_amd.PagedKVCache(12, P, hkv, D, 2, 6, DTYPES[kind], *([0.02] * 2 if kind == "fp8" else [1.0] * 2))
    for step in range(3):
        (q2, k2, v2), _ = make_heads(rng, 2, (hq, hkv, hkv), False)
        q.copy_(q2), k.copy_(k2), v.copy_(v2)
        graph.replay()
        torch.cuda.synchronize()
        # The same appends, eagerly, on a cache of their own (a replay keeps the scale that the one before raised).
        if step == 0:
            for _ in range(2):
                eager.admit()
            eager.append_rope([0], [20], k0, v0, rope)
            want = eager.append_rope([0, 1], [1, 1], k2, v2, rope, q=q2)
            a, b = (cache_view(c, kind, 12, hkv, P) for c in (cache, eager))
            for s, n in ((0, 21), (1, 1)):
                for x, y in zip(stored(*a, cache.block_table(s), n, P, 1.0), stored(*b, eager.block_table(s), n, P, 1.0)):
                    assert np.array_equal(x, y)
        else:
            want, _ = pa_amd.norm_rope(q2, None, torch.tensor([20, 0], dtype=torch.int32, device="cuda"), rope)
            got = stored(*cache_view(cache, kind, 12, hkv, P), cache.block_table(1), 1, P, 0.02 if kind == "fp8" else 1.0)
            vv = v2[1].float().cpu().numpy().astype(np.float64)
            assert np.all(np.abs(got[1][0] - vv) <= np.abs(vv) * 2.0 ** -4 + 2.0 ** -6)
        assert np.array_equal(bits(out), bits(want))
    cache.close()
    eager.close()


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("entries,empty", [(3, False), (65, True), (200, False), (4500, True)])
def test_append_rope_many_entries(kind, entries, empty):
    """Entries are found among many, evenly spread or not (empty ones, one long one among single tokens)."""
    import torch
    rng = np.random.default_rng(entries)
    hkv, P, rows = 1, 16, entries
    counts = np.ones(entries, int)
    if empty:
        counts[rng.random(entries) < 0.5] = 0
    counts[entries // 3] = 100
    starts = rng.integers(0, 16, entries)
    cols = 8
    table = np.arange(rows * cols, dtype=np.int32)[::-1].reshape(rows, cols).copy()
    begin = np.concatenate([[0], np.cumsum(counts)])
    n = int(begin[-1])
    kb, vb = normal_f16(rng, (n, hkv, D)), normal_f16(rng, (n, hkv, D))
    eb = torch.float16 if kind == "fp16" else torch.uint8
    k_cache, v_cache = (torch.zeros((rows * cols, hkv, P, D), dtype=eb, device="cuda") for _ in range(2))
    scales = pa_amd.alloc_kv_scales(rows * cols, hkv, P) if kind == "block" else None
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    pa_amd.append_rope(None, half(kb), half(vb), k_cache, v_cache, to_device(table), dev(begin), dev(starts), kv_scales=scales)
    torch.cuda.synchronize()
    e = np.repeat(np.arange(entries), counts)
    pos = starts[e] + np.arange(n) - begin[e]
    page, slot = table[e, pos // P], pos % P
    for t, b in ((k_cache, kb), (v_cache, vb)):
        got = t.cpu()
        if kind == "fp16":
            host = got.view(torch.int16).numpy().view(np.uint16)
            assert np.array_equal(host[page, :, slot], b)
        elif kind == "fp8":
            host = got.numpy()
            assert np.array_equal(host[page, :, slot], nt.e4m3_encode(nt.f16(b)))
        else:
            host = got.numpy()
            sc = scales.cpu().numpy()[page, :, slot // 16, 0 if t is k_cache else 1].astype(int) - 127
            val = nt.e4m3(host[page, :, slot]) * 2.0 ** sc[..., None]
            assert np.all(np.abs(val - nt.f16(b)) <= np.maximum(np.abs(nt.f16(b)) * 2.0 ** -4, 2.0 ** (sc[..., None] - 10.0)))
        assert int((host != 0).any(axis=(1, 3)).sum()) == n   # one row each, no other


@pytest.mark.parametrize("kind", CACHES)
def test_append_rope_several_axes(binding, kind):
    """Image tokens: three positions each, in a cache at places of its own."""
    import torch
    rng = np.random.default_rng(3)
    n, hq, hkv, P, pages = 50, 4, 2, 16, 6
    cache = Paged(rng, kind, pages, hkv, P)
    cache.begin()
    axis = np.repeat([0, 1, 2], [16, 24, 24])
    rope = pa_amd.Rope(nt.freqs(128), axes=axis)
    assert rope.num_axes == 3
    pos = rng.integers(0, 4096, (n, 3))
    table = rng.permutation(pages)[:4].astype(np.int32)
    (q, k, v), (qb, kb, vb) = make_heads(rng, n, (hq, hkv, hkv), True)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    args = (to_device(table[None]), dev([0, n]), dev([7]), rope)
    with pytest.raises(ValueError, match="axes"):
        pa_amd.append_rope(q, k, v, *cache.dev, *args, **cache.args())
    qo = pa_amd.append_rope(q, k, v, *cache.dev, *args, positions=dev(pos), **cache.args())
    ref, mag = nt.norm_rotate(nt.f16(kb), None, 0, pos, nt.freqs(128), axis)
    cache.append(ref, mag, vb, 7, table)
    cache.check()
    check_rows(bits(qo), *nt.norm_rotate(nt.f16(qb), None, 0, pos, nt.freqs(128), axis))


@pytest.mark.parametrize("kind", CACHES)
def test_append_rope_past_4_gib(kind):
    """Pages whose offsets pass 32 bits, in bytes and in elements."""
    import torch
    rng = np.random.default_rng(4)
    hkv, P = 8, 128
    eb = 2 if kind == "fp16" else 1
    pages = (5 << 30) // (hkv * P * D * eb)
    dt = torch.float16 if kind == "fp16" else torch.uint8
    k_cache, v_cache = (torch.empty((pages, hkv, P, D), dtype=dt, device="cuda") for _ in range(2))
    scales = pa_amd.alloc_kv_scales(pages, hkv, P) if kind == "block" else None
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    n = 2 * P + 9
    kb, vb = normal_f16(rng, (n, hkv, D)), normal_f16(rng, (n, hkv, D))
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    pa_amd.append_rope(None, half(kb), half(vb), k_cache, v_cache, table, dev([0, n]), dev([0]), kv_scales=scales)
    d = pa_amd.Decoder(8, hkv, D, P, kind != "fp16", **(dict(block_scales=True) if kind == "block" else {}))
    lens = torch.tensor([n], dtype=torch.int32)
    d.plan(lens)
    qb = normal_f16(rng, (1, 8, D))
    out = d.run(half(qb), k_cache, v_cache, table, lens.cuda(), 1.0, 1.0, **(dict(kv_scales=scales) if kind == "block" else {}))
    torch.cuda.synchronize()
    pg = np.array([pages - 1, 0, pages - 2])
    held = [t[torch.from_numpy(pg).cuda()].cpu() for t in (k_cache, v_cache)]
    sc = None if scales is None else scales[torch.from_numpy(pg).cuda()].cpu().numpy()
    pools = [t.view(torch.int16).numpy().view(np.uint16) if kind == "fp16" else t.numpy() for t in held]
    k, v = stored(pools, sc, [0, 1, 2], n, P, 1.0)
    for got, b in ((k, kb), (v, vb)):
        want = nt.f16(b)
        tol = 0 if kind == "fp16" else np.abs(want) * 2.0 ** -4 + 2.0 ** -10
        assert np.all(np.abs(got - want) <= tol)
    ref, weight, big = nt.attention(nt.f16(qb[0]), k, v)
    assert np.all(np.abs(out[0].double().cpu().numpy() - ref) <= nt.attention_tol(ref, weight, big))


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("lead,tail", [(0, 7), (5, 0), (3, 40)])
def test_append_rope_padded(kind, lead, tail):
    """Tokens before the first entry and after the last are in none: left out, their q is not."""
    import torch
    rng = np.random.default_rng(lead + tail)
    hq, hkv, P, pages = 4, 2, 16, 8
    cache = Paged(rng, kind, pages, hkv, P)
    cache.begin()
    counts, starts = [1, 20, 1], [13, 15, 0]
    begin = lead + np.concatenate([[0], np.cumsum(counts)])
    n = int(begin[-1]) + tail
    table = np.array([[0, 1, 2], [3, 4, 5], [6, 7, 7]], np.int32)
    (q, k, v), (qb, kb, vb) = make_heads(rng, n, (hq, hkv, hkv), True)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    qo = pa_amd.append_rope(q, k, v, *cache.dev, to_device(table), dev(begin), dev(starts), **cache.args())
    for e, (c, s) in enumerate(zip(counts, starts)):
        part = slice(begin[e], begin[e] + c)
        cache.append(nt.f16(kb[part]), np.abs(nt.f16(kb[part])), vb[part], s, table[e])
    cache.check()
    assert np.array_equal(bits(qo), qb)


def test_norm_rope_replayed():
    """Captured, every replay turns what is then in q, k and positions, beside eager calls on the same Rope."""
    import torch
    rng = np.random.default_rng(6)
    rope = pa_amd.Rope(nt.freqs(128))
    (q, k), _ = make_heads(rng, 9, (8, 2), False)
    pos = torch.zeros(9, dtype=torch.int32, device="cuda")
    w, wf = weights(rng, True)
    pa_amd.norm_rope(q, k, pos, rope)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = pa_amd.norm_rope(q, k, pos, rope, q_weight=w, k_weight=w)
    for step in range(4):
        (q2, k2), (qb, kb) = make_heads(rng, 9, (8, 2), False)
        p = rng.integers(0, 9999, 9)
        q.copy_(q2), k.copy_(k2), pos.copy_(torch.from_numpy(p.astype(np.int32)))
        graph.replay()
        eager = pa_amd.norm_rope(q2, k2, pos, rope, q_weight=w, k_weight=w)
        torch.cuda.synchronize()
        for got, same, b in ((qo, eager[0], qb), (ko, eager[1], kb)):
            assert np.array_equal(bits(got), bits(same))
            check_rows(bits(got), *nt.norm_rotate(nt.f16(b), wf, float(np.float32(1e-6)), p, nt.freqs(128)))
