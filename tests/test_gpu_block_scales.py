"""GPU tests of the block-scaled E4M3 cache: what its appends store (bit for bit against a plain model of its history) and
attention over it, alone and in whole serving steps, against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

import new_tokens as nt
import pa_amd
from helpers import D, normal_f16, to_device
from test_gpu_new_tokens import CACHES, DTYPES, bits, cache_view, half, make_heads, stored, weights

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def dev(a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def hard_values(rng, n, hkv):
    """fp16 rows over the whole range: zeros, subnormals, the largest values, infinities, NaN of both signs."""
    x = (rng.standard_normal((n, hkv, D)) * 2.0 ** rng.integers(-22, 14, (n, hkv, 1))).astype(np.float16)
    x[rng.random((n, hkv)) < 0.1] = 0
    x[rng.random((n, hkv)) < 0.03] = 65504
    some = rng.random(x.shape)
    x[some < 0.002] = np.inf
    x[(some > 0.002) & (some < 0.004)] = -np.inf
    b = x.view(np.uint16)
    b[(some > 0.004) & (some < 0.006)] = 0x7E01
    b[(some > 0.006) & (some < 0.008)] = 0xFE01
    return b


@pytest.mark.parametrize("P", [8, 16, 24, 48, 128])
@pytest.mark.parametrize("steps", [[40], [1] * 19, [5, 11, 1, 1, 30, 2], [15, 2, 100]])
@pytest.mark.parametrize("hard", [False, True], ids=["normal", "hard"])
def test_blocks_hold_their_history(P, steps, hard):
    """Rows without a rotation are fp16 values: codes and scales equal the plain model's, whatever the steps that a
    block fills in."""
    import torch
    rng = np.random.default_rng(P + len(steps))
    hkv, n = 3, sum(steps)
    cols = -(-n // P)
    table = rng.permutation(cols + 2)[:cols].astype(np.int32)
    start_codes = rng.integers(0, 256, (2, cols + 2, hkv, P, D), dtype=np.uint8)
    sc = rng.integers(0, 256, (cols + 2, hkv, P // nt.block_tokens(P), 2), dtype=np.uint8)   # of pages' earlier owners
    pools = [nt.BlockPool(start_codes[j], sc[..., j]) for j in range(2)]
    k_cache, v_cache, scales = (to_device(a) for a in (start_codes[0], start_codes[1], sc))
    at = 0
    for c in steps:
        if hard:
            kb, vb = hard_values(rng, c, hkv), hard_values(rng, c, hkv)
        else:
            kb, vb = normal_f16(rng, (c, hkv, D)), normal_f16(rng, (c, hkv, D))
        pa_amd.append_rope(None, half(kb), half(vb), k_cache, v_cache, to_device(table[None]), dev([0, c]), dev([at]),
                           kv_scales=scales)
        for pool, b in zip(pools, (kb, vb)):
            pool.append(nt.f16(b), at, table)
        at += c
        torch.cuda.synchronize()
        got = scales.cpu().numpy()
        for j, (pool, t) in enumerate(zip(pools, (k_cache, v_cache))):
            assert np.array_equal(got[..., j].astype(int) - 127, pool.exps)
            assert np.array_equal(t.cpu().numpy(), pool.codes)


def paged(rng, lens, hkv, P, spread=3, hot=None):
    """A block-scaled cache of sequences of these lengths: codes everywhere (the rows behind a sequence hold NaN), scale
    exponents over `spread` around one of each sequence; returns the device's and the plain values."""
    pages_of = [-(-n // P) for n in lens]
    total = sum(pages_of) + 2
    b = nt.block_tokens(P)
    codes = rng.integers(0, 0x78, (2, total, hkv, P, D), dtype=np.uint8) | (rng.integers(0, 2, (2, total, hkv, P, D), dtype=np.uint8) << 7)
    exps = rng.integers(-9, -9 + spread, (total, hkv, P // b, 2))
    if hot is not None:
        exps[..., hot[0]] = hot[1]
    perm = rng.permutation(total).astype(np.int32)
    table = np.full((len(lens), max(pages_of)), perm[-1], np.int32)
    at = 0
    for r, (n, c) in enumerate(zip(lens, pages_of)):
        table[r, :c] = perm[at:at + c]
        at += c
        if n % P:
            codes[:, table[r, c - 1], :, n % P:] = 0x7F
    values = [nt.e4m3(codes[j]) * np.repeat(2.0 ** exps[..., j], b, axis=2)[..., None] for j in range(2)]
    dk, dv = (to_device(codes[j]) for j in range(2))
    scales = to_device((exps + 127).astype(np.uint8))
    rows = []
    for r, n in enumerate(lens):
        t = np.arange(n)
        rows.append([v[table[r, t // P], :, t % P] for v in values])
    return dk, dv, scales, to_device(table), rows


def check_decode(out, qb, rows):
    got = out.double().cpu().numpy()
    for r, (k, v) in enumerate(rows):
        ref, weight, big = nt.attention(nt.f16(qb[r]), k, v)
        err = np.abs(got[r] - ref)
        tol = nt.attention_tol(ref, weight, big)
        assert np.all(err <= tol), (r, float((err / tol).max()))


@pytest.mark.parametrize("P", [8, 16, 24, 32, 48, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (4, 2), (32, 8), (8, 1)])
def test_decode_block_scales(P, hq, hkv):
    """Ragged rows: one token, a block less and more one, several segments."""
    import torch
    rng = np.random.default_rng(P * 100 + hq)
    lens = [1, 15, 16, 17, 33, 200, 8, 777]
    dk, dv, scales, table, rows = paged(rng, lens, hkv, P)
    qb = normal_f16(rng, (len(lens), hq, D))
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    lt = torch.tensor(lens, dtype=torch.int32)
    d.plan(lt)
    out = d.run(half(qb), dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=scales)
    torch.cuda.synchronize()
    check_decode(out, qb, rows)
    # Both bindings and any grid: within the same bounds; the same plan the same bits.
    from pa_amd.decoder import Decoder
    for ctas in (0, 3):
        e = Decoder(hq, hkv, D, P, True, True)
        e.plan(lt, ctas)
        o = e.run(half(qb), dk, dv, table, lt.cuda(), 1.0, 1.0, scales)
        torch.cuda.synchronize()
        check_decode(o, qb, rows)
        if ctas == 0:
            assert torch.equal(o, out)


@pytest.mark.parametrize("lens,hq,hkv,P", [([5000], 32, 8, 16), ([30001, 3], 8, 1, 24), ([1] * 70, 16, 2, 16)])
def test_decode_block_scales_merges(lens, hq, hkv, P):
    """Rows over many blocks (the merge kernel), over few (merged in the split kernel), and many short ones."""
    import torch
    rng = np.random.default_rng(len(lens))
    dk, dv, scales, table, rows = paged(rng, lens, hkv, P, spread=2)
    qb = normal_f16(rng, (len(lens), hq, D))
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    lt = torch.tensor(lens, dtype=torch.int32)
    d.plan(lt)
    out = d.run(half(qb), dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=scales)
    torch.cuda.synchronize()
    check_decode(out, qb, rows)


@pytest.mark.parametrize("which,exp", [(0, -32), (1, -32), (1, -20), (1, 7), (0, 1)])
def test_decode_block_scales_extremes(which, exp):
    """Keys or values of the smallest and largest scales that appends choose."""
    import torch
    rng = np.random.default_rng(77)
    lens, hq, hkv, P = [100, 17], 16, 4, 16
    dk, dv, scales, table, rows = paged(rng, lens, hkv, P, hot=(which, exp))
    qb = (rng.standard_normal((2, hq, D)) * 0.02).astype(np.float16).view(np.uint16)
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    lt = torch.tensor(lens, dtype=torch.int32)
    d.plan(lt)
    out = d.run(half(qb), dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=scales)
    torch.cuda.synchronize()
    check_decode(out, qb, rows)


@pytest.mark.parametrize("nan", [False, True])
def test_decode_block_scales_of_one_are_the_per_tensor_kernel(nan):
    """Scales of 1 and a per-tensor scale of 1: the same values, the same bits (NaN keys among them: NaN rows)."""
    import torch
    rng = np.random.default_rng(5)
    lens, hq, hkv, P = [300, 1, 64], 32, 8, 16
    dk, dv, scales, table, _ = paged(rng, lens, hkv, P)
    if nan:
        dk[dk >= 0x80] -= 0x40   # 0xbf, a moderate value, becomes 0x7f, a NaN
    else:
        dk &= 0xBF               # smaller codes: scores stay moderate
    scales.fill_(127)
    q = half((rng.standard_normal((3, hq, D)) * 0.01).astype(np.float16).view(np.uint16))
    lt = torch.tensor(lens, dtype=torch.int32)
    outs = []
    for block in (False, True):
        d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=block)
        d.plan(lt)
        outs.append(d.run(q, dk, dv, table, lt.cuda(), 1.0, 1.0, **(dict(kv_scales=scales) if block else {})))
    torch.cuda.synchronize()
    assert torch.isfinite(outs[0]).all() != nan and torch.equal(*(o.view(torch.int16) for o in outs))


def test_decoder_refuses_scales():
    import torch
    rng = np.random.default_rng(6)
    dk, dv, scales, table, _ = paged(rng, [20], 2, 16)
    lt = torch.tensor([20], dtype=torch.int32)
    q = half(normal_f16(rng, (1, 4, D)))
    from pa_amd.decoder import Decoder
    for cls in (pa_amd.Decoder, Decoder):
        d = cls(4, 2, D, 16, True, block_scales=True)
        d.plan(lt)
        for bad in (None, scales[:-1], scales.float(), scales[..., :1], scales.cpu(), scales.transpose(0, 1)):
            with pytest.raises(RuntimeError):
                d.run(q, dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=bad)
        e = cls(4, 2, D, 16, True)
        e.plan(lt)
        with pytest.raises(RuntimeError, match="block_scales"):
            e.run(q, dk, dv, table, lt.cuda(), 1.0, 1.0, kv_scales=scales)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("P", [16, 24])
def test_serving_steps(kind, P):
    """The operators as a server runs them: prompts and decode steps go in with append_rope (q beside them), every step
    is planned and decoded; a sequence leaves, its pages go to another (whose blocks start anew). Every output against
    attention in 64 bits over what the cache holds, and what it holds against the rotated keys."""
    import torch
    rng = np.random.default_rng(31 + P)
    hq, hkv, slots, cols = 8, 2, 4, 12
    scale = 6.0 / 448 if kind == "fp8" else 1.0
    pages = 26
    cache = pa_amd.PagedKVCache(pages, P, hkv, D, slots, cols, DTYPES[kind], scale, scale)
    cache.shuffle_free_pages(2)
    fr = nt.freqs(96)
    rope = pa_amd.Rope(fr)
    wq, wqf = weights(rng, True)
    wk, wkf = weights(rng, True)
    kept: dict[int, list] = {}
    joins = {0: [40, 1], 1: [100], 3: [17], 4: [60]}
    for step in range(7):
        if step == 4:
            gone = next(iter(kept))
            cache.release(gone)
            del kept[gone]
        sl, counts = list(kept), [1] * len(kept)
        for n in joins.get(step, []):
            s = cache.admit()
            assert s >= 0
            kept[s] = []
            sl.append(s)
            counts.append(n)
        n = sum(counts)
        (q, k, v), (qb, kb, vb) = make_heads(rng, n, (hq, hkv, hkv), True)
        place = np.concatenate([np.arange(c) + len(kept[s]) for s, c in zip(sl, counts)])
        out_q = cache.append_rope(sl, counts, k, v, rope, q=q, q_weight=wq, k_weight=wk)
        ref, mag = nt.norm_rotate(nt.f16(kb), wkf, float(np.float32(1e-6)), place, fr)
        lo, last = 0, []
        for s, c in zip(sl, counts):
            kept[s] += [(ref[i], mag[i], nt.f16(vb[i])) for i in range(lo, lo + c)]
            lo += c
            last.append(lo - 1)
        # The last token of each sequence attends.
        qd = out_q[torch.tensor(last, device="cuda")].contiguous()
        out = torch.empty_like(qd)
        cache.plan(sl, hq)
        cache.run(qd, out)
        torch.cuda.synchronize()
        view = cache_view(cache, kind, pages, hkv, P)
        rows = []
        for s in sl:
            L = len(kept[s])
            assert cache.seq_len(s) == L
            rows.append(stored(*view, cache.block_table(s), L, P, scale if kind == "fp8" else 1.0))
            for j, col in ((0, 0), (1, 2)):
                want = np.array([t[col] for t in kept[s]])
                m = np.array([t[1] for t in kept[s]]) if j == 0 else np.abs(want)
                if kind == "fp16":
                    tol = nt.f16_tol(want, m)
                else:
                    step_of = scale
                    if kind == "block":
                        t = np.arange(L)
                        b = nt.block_tokens(P)
                        e = view[1][np.asarray(cache.block_table(s))[t // P], :, t % P // b, j].astype(int) - 127
                        step_of = 2.0 ** e[..., None]
                    tol = nt.e4m3_tol(want, m, step_of) + (step_of * 2.0 ** -10 if kind == "block" else 0.0)
                assert np.all(np.abs(rows[-1][j] - want) <= tol)
        check_decode(out, bits(qd), rows)
    cache.close()


def test_block_cache_on_another_stream():
    """Appends, plan and decode queued on a side stream while the default stream works; releases in between."""
    import torch
    rng = np.random.default_rng(41)
    hq, hkv, P = 8, 2, 16
    cache = pa_amd.PagedKVCache(20, P, hkv, D, 2, 10, pa_amd.FP8_E4M3_BLOCK)
    rope = pa_amd.Rope(nt.freqs(128))
    side = torch.cuda.Stream()
    busy = torch.zeros(1 << 24, device="cuda")
    for turn in range(3):
        s = cache.admit()
        (q, k, v), (qb, kb, vb) = make_heads(rng, 50, (hq, hkv, hkv), True)
        torch.cuda.synchronize()
        for _ in range(5):
            busy += 1
        with torch.cuda.stream(side):
            qo = cache.append_rope([s], [50], k, v, rope, q=q)
            qd = qo[49:].contiguous()
            out = torch.empty_like(qd)
            cache.plan([s], hq)
            cache.run(qd, out)
        side.synchronize()
        rows = [stored(*cache_view(cache, "block", 20, hkv, P), cache.block_table(s), 50, P, 1.0)]
        check_decode(out, bits(qd), rows)
        ref, _ = nt.norm_rotate(nt.f16(kb), None, 0, np.arange(50), nt.freqs(128))
        assert np.abs(rows[0][0] - ref).max() < np.abs(ref).max() * 2.0 ** -4
        cache.release(s)
    cache.close()


def test_step_replayed_over_a_caller_s_cache():
    """Append and attention of one step in a graph, over pools of the caller's: every replay stores the tokens then in
    k and v and attends with the q then there; eager steps on a cache of their own between the replays."""
    import torch
    rng = np.random.default_rng(51)
    hq, hkv, P, pages, m = 8, 2, 16, 12, 3
    lens = [17, 5, 40]                                 # with the step's token
    table = rng.permutation(pages).astype(np.int32).reshape(m, 4)[:, :3].copy()
    rope = pa_amd.Rope(nt.freqs(128))
    dt = to_device(table)
    begin, starts = dev(list(range(m + 1))), dev([n - 1 for n in lens])
    lt = torch.tensor(lens, dtype=torch.int32)
    lens_dev = lt.cuda()

    def fresh():
        k_cache, v_cache = (torch.zeros((pages, hkv, P, D), dtype=torch.uint8, device="cuda") for _ in range(2))
        return k_cache, v_cache, pa_amd.alloc_kv_scales(pages, hkv, P)

    (pk, pv), _ = make_heads(rng, sum(lens) - m, (hkv, hkv), False)
    caches = [fresh(), fresh()]
    for c in caches:
        pa_amd.append_rope(None, pk, pv, c[0], c[1], dt, dev(np.concatenate([[0], np.cumsum([n - 1 for n in lens])])),
                           dev([0] * m), rope, kv_scales=c[2])
    d = pa_amd.Decoder(hq, hkv, D, P, True, block_scales=True)
    d.plan(lt)
    (q, k, v), _ = make_heads(rng, m, (hq, hkv, hkv), False)

    def step(c, q, k, v):
        qo = pa_amd.append_rope(q, k, v, c[0], c[1], dt, begin, starts, rope, kv_scales=c[2])
        return d.run(qo, c[0], c[1], dt, lens_dev, 1.0, 1.0, kv_scales=c[2])

    step(caches[1], q, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], q, k, v)
    step(caches[0], q, k, v)   # what the eager cache has seen
    for _ in range(4):
        (q2, k2, v2), _ = make_heads(rng, m, (hq, hkv, hkv), False)
        q.copy_(q2), k.copy_(k2), v.copy_(v2)
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1], q2, k2, v2)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(out).all()
        for a, b in zip(*caches):
            assert torch.equal(a, b)
