"""GPU tests of the numbers that attention of drafted tokens and rows read back stand for, where they are very small or
very large."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import pa_amd
from drafts import D, Cache, attention, random_tree, seen_of
from test_gpu_drafts import begins, check_attention, cols_for, ints, run_attention

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


# Exponents of K's and V's scales (of 448 2^k, V's largest is an fp16 value up to k = 7), and a softmax scale at which
# scores are of order one.
RANGES = {"smallest": ((-32, -26), (-32, -20), 2.0 ** 20), "largest": ((3, 9), (0, 8), 2.0 ** -15),
          "all": ((-32, 9), (-32, 8), 2.0 ** -14)}


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("which", list(RANGES))
@pytest.mark.parametrize("entries,chain", [([(0, 3), (70, 9)], False), ([(200, 40)], True), ([(3000, 100)], False)])
def test_block_scales_over_their_range(which, entries, chain, page):
    """K's scales multiply scores in 32 bits; V's rows are fp16, within 2^-25 below 2^-14."""
    (k0, k1), (v0, v1), scale = RANGES[which]
    cache = Cache("block", page, 2, len(entries), cols_for(entries, page), seed=page)
    r = np.random.default_rng(page)
    shape = cache.scales.shape[:-1]
    cache.scales[..., 0] = r.integers(127 + k0, 127 + k1, shape)
    cache.scales[..., 1] = r.integers(127 + v0, 127 + v1, shape)
    if which != "smallest":   # keys past fp16, 448 * 2^8
        cache.kv[0].reshape(-1)[::4001] = 0x7e
        cache.scales[::3, ..., 0] = 135
    trees = None if chain else [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    out, q = run_attention(cache, entries, 8, trees, sm_scale=scale)
    check_attention(cache, entries, 8, trees, out, q, scale=scale)


def test_decode_and_attention_agree_on_small_keys():
    """One token over keys near 2^-30, as the decode has it."""
    hq, hkv, page, lens = 8, 2, 16, [300, 77]
    cache = Cache("block", page, hkv, 2, cols_for([(n, 0) for n in lens], page), seed=1)
    cache.scales[..., 0] = np.random.default_rng(0).integers(92 + 3, 92 + 8, cache.scales.shape[:-1])
    k, v, table, scales = cache.device()
    q = torch.from_numpy((np.random.default_rng(1).standard_normal((2, hq, D)) * 6e4 / 5).astype(np.float16)).cuda()
    q_scale = 2.0 ** 7 * D ** 0.5                     # (the decode's softmax scale is 1 / sqrt(128): k_scale takes the rest)
    dec = pa_amd.Decoder(hq, hkv, D, page, True, block_scales=True)
    dec.plan(torch.tensor(lens, dtype=torch.int32))
    one = dec.run(q, k, v, table, ints(lens), q_scale, 1.0, kv_scales=scales)
    same = pa_amd.tree_attention(q, k, v, table, begins([1, 1]), ints(n - 1 for n in lens), k_scale=q_scale, kv_scales=scales)
    for e, n in enumerate(lens):
        K, V = (cache.rows(j, e, 0, n) for j in range(2))
        ref, tol = attention(q[e:e + 1].double().cpu().numpy(), K, V, np.ones((1, n), bool), q_scale / D ** 0.5)
        for got in (one, same):
            assert (np.abs(got[e].double().cpu().numpy() - ref[0]) <= tol[0]).all(), e


@pytest.mark.parametrize("kind", ["fp16", "fp8"])
@pytest.mark.parametrize("low", [-14.5, -17.5])
def test_tails(kind, low):
    """A place of score 0 and 99999 of `low`: probabilities that are subnormal in fp16 and a twentieth of the sum."""
    n = 100_000
    cache = Cache(kind, 16, 1, 1, n // 16, seed=3, k_scale=2.0 ** -6, v_scale=2.0 ** -8)
    if kind == "fp16":
        cache.kv[0][:] = 0
        cache.kv[0][..., 0] = low / 16
        cache.kv[1] = np.abs(cache.kv[1])
    else:
        cache.kv[0][:] = 0
        cache.kv[0][..., 0] = {-14.5: 0xe7, -17.5: 0xe9}[low]      # -60 and -72, 2^-6 of which times 16 is near `low`
        cache.kv[1] &= 0x7f
    page = cache.table[0, 0]
    cache.kv[0][page, :, 0, 0] = 0
    cache.kv[1][page, :, 0] = 0
    q = np.zeros((1, 2, D), np.float16)
    q[..., 0] = 16.0
    out, _ = run_attention(cache, [(n - 1, 1)], 2, None, q=q, sm_scale=1.0)
    check_attention(cache, [(n - 1, 1)], 2, None, out, q, scale=1.0)


def odd_reference(q, k, v, seen, scale):
    """attention() with values that are not finite: their sum, in the dims where a token sees some, whatever their
    weight; elsewhere they count as 0."""
    fine = np.isfinite(v)
    ref, tol = attention(q, k, np.where(fine, v, 0.0), seen, scale)
    group = q.shape[1] // k.shape[1]
    odd = np.where(fine, 0.0, v)
    with np.errstate(invalid="ignore"):
        sums = np.stack([odd[m].sum(0) for m in seen])               # [n, hkv, 128]
    sums = np.repeat(sums, group, axis=1)
    return np.where(sums == 0, ref, sums), tol


def check_odd(cache, entries, hq, trees, out, q, scale):
    got, at = out.double().cpu().numpy(), 0
    for e, (start, n) in enumerate(entries):
        k, v = (cache.rows(j, e, 0, start + n) for j in range(2))
        ref, tol = odd_reference(q[at:at + n].astype(np.float64), k, v, seen_of(start, n, None if trees is None else trees[e]), scale)
        fine, mine = np.isfinite(ref), got[at:at + n]
        assert not fine.all()
        np.testing.assert_array_equal(mine[~fine], ref[~fine])
        assert (np.abs(mine[fine] - ref[fine]) <= tol[fine]).all(), e
        at += n


# Entries: in one tile, cut over many blocks, beside one that makes the tiles larger.
@pytest.mark.parametrize("entries", [[(300, 3)], [(9000, 20)], [(700, 4), (50, 120)], [(1000, 150)]])
@pytest.mark.parametrize("kind,page", [("fp16", 16), ("fp16", 5), ("fp8", 16), ("block", 24)])
@pytest.mark.parametrize("peak", [0.0, 400.0])
def test_values_that_are_not_finite_anywhere(kind, page, entries, peak):
    """Infinities and NaN at early places, which every token sees, and among an entry's own: the tokens that see one have
    it, of whatever weight (a peak of 400 above the other scores leaves them none), its other dims and the other
    tokens are as they were."""
    cache = Cache(kind, page, 2, len(entries), cols_for(entries, page), seed=8)
    put = {"fp16": [np.inf, -np.inf, np.nan], "fp8": [0x7f, 0xff], "block": [0x7e, 0xfe, 0x7f]}[kind]
    for e, (start, n) in enumerate(entries):
        places = (0, 17, 40, start // 2, start - 1, start, start + n // 2, start + n - 1)
        if kind == "block":                          # 448 * 2^8 is past fp16: infinite
            for pos in places:
                p, s = cache.table[e, pos // page], pos % page
                cache.scales[p, :, s // 8, 1] = 135
                cache.kv[1][p, :, s // 8 * 8:s // 8 * 8 + 8] &= 0xf7   # (240 at most)
        for i, pos in enumerate(places):
            p, s = cache.table[e, pos // page], pos % page
            cache.kv[1][p, :, s, 4 * i:4 * i + 6] = put[i % len(put)]
    n = sum(m for _, m in entries)
    q = np.random.default_rng(0).standard_normal((n, 8, D)).astype(np.float16)
    if peak:   # dim 0 of K: one place (of the second half, say) that all rows find far above the others
        q[..., 0] = 16.0
        for e, (start, m) in enumerate(entries):
            for pos in range(start + m):
                cache.kv[0][cache.table[e, pos // page], :, pos % page, 0] = 0
            p, s = cache.table[e, 30 // page], 30 % page
            one = {"fp16": np.float16(peak), "fp8": 0x7e, "block": 0x7e}[kind]
            cache.kv[0][p, :, s, 0] = one
            if kind == "block":
                cache.scales[p, :, s // 8, 0] = 127
    scale = 1.0 if peak else 0.1
    if kind == "fp8" and peak:
        cache.k_scale = 1.0
    trees = [random_tree(np.random.default_rng(i), m) for i, (_, m) in enumerate(entries)]
    for t in (trees, None):
        out, _ = run_attention(cache, entries, 8, t, q=q, sm_scale=scale)
        values = Cache.rows
        if kind == "block":   # (as the kernel has them: infinite past fp16)
            def values(self, j, row, lo, hi, rows=Cache.rows):
                x = rows(self, j, row, lo, hi)
                return np.where(np.abs(x) > 65504, np.sign(x) * np.inf, x) if j else x
        keep, Cache.rows = Cache.rows, values
        try:
            check_odd(cache, entries, 8, t, out, q, scale)
        finally:
            Cache.rows = keep


@pytest.mark.parametrize("start", [40, 5000])
def test_a_query_that_is_not_a_number_over_values_that_are_not(start):
    """It has NaN in every dim; the others are as ever, in a captured call, too, once the value is there and once it is
    gone."""
    n, hq = 20, 8
    cache = Cache("fp16", 16, 2, 1, cols_for([(start, n)], 16), seed=5)
    k, v, table, _ = cache.device()
    q = np.random.default_rng(0).standard_normal((n, hq, D)).astype(np.float16)
    plain = q.copy()
    q[7, 2, 9] = np.nan
    dq, tb, starts = torch.from_numpy(q).cuda(), begins([n]), ints([start])
    out = torch.empty_like(dq)
    pa_amd.tree_attention(dq, k, v, table, tb, starts, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pa_amd.tree_attention(dq, k, v, table, tb, starts, out=out)
    page, slot = int(cache.table[0, 20 // 16]), 20 % 16
    for x in (np.inf, 1.0, np.nan, -np.inf, 2.0):
        cache.kv[1][page, :, slot, 30:40] = x
        v[page, :, slot, 30:40] = float(x)
        g.replay()
        torch.cuda.synchronize()
        got = out.float().cpu().numpy()
        assert np.isnan(got[7, 2]).all()
        kk, vv = (cache.rows(j, 0, 0, start + n) for j in range(2))
        ref, tol = odd_reference(plain.astype(np.float64), kk, vv, seen_of(start, n, None), D ** -0.5)
        got[7, 2], fine = ref[7, 2], np.isfinite(ref)
        np.testing.assert_array_equal(got[~fine], ref[~fine])
        assert (np.abs(got[fine] - ref[fine]) <= tol[fine]).all()


@pytest.mark.parametrize("scale", [2.0 ** 120, 2.0 ** -100, 1.7e38, 3e-38])
def test_read_cache_of_large_and_small_scales(scale):
    """code * scale in 32 bits, rounded once: a block's scale times the cache's may be past fp32 where its codes'
    values are not."""
    cache = Cache("block", 16, 2, 1, 4, seed=2)
    r = np.random.default_rng(3)
    shape = cache.scales.shape
    cache.scales = np.where(r.random(shape) < 0.5, 135, 95).astype(np.uint8)
    cache.kv = [r.integers(0, 256, x.shape).astype(np.uint8) for x in cache.kv]
    for x in cache.kv:
        x[..., ::3] &= 0x87                          # zeros and subnormals among them
    k, v, table, scales = cache.device()
    got = pa_amd.read_cache(k, v, table, begins([64]), ints([0]), 64, dtype=torch.float32, k_scale=scale, v_scale=scale,
                            kv_scales=scales)
    for j in range(2):
        x = cache.rows(j, 0, 0, 64)
        with np.errstate(over="ignore", invalid="ignore"):
            want = x.astype(np.float32) * np.float32(scale)
        np.testing.assert_array_equal(got[j].cpu().numpy(), want)
