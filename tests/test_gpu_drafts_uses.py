"""GPU tests of uses of the drafted-token operators that their documentation allows: a whole step of drafted tokens beside
appends and decodes, caches and rows whose offsets pass 32 bits, graphs that share memory, odd scales and operands."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import drafts
import new_tokens as nt
import pa_amd
from drafts import D, Cache, attention, random_tree, seen_of
from helpers import to_device
from test_gpu_drafts import begins, check_attention, cols_for, ints, run_attention

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def scales_of(kind):
    return {"k_scale": 0.02, "v_scale": 0.03} if kind == "fp8" else {}


@pytest.mark.parametrize("kind,page", [("fp16", 16), ("fp8", 16), ("block", 16), ("block", 24), ("fp16", 5)])
def test_a_step_of_drafted_tokens(kind, page):
    """Prompts appended, trees of drafted tokens appended behind them, attention of the trees, the accepted branch kept,
    the next token appended and decoded: each against the rows that read_cache gives, and the kept rows against a cache
    that only ever saw the accepted tokens."""
    r = np.random.default_rng(7)
    hq, hkv, starts, m, cols = 8, 2, [70, 13, 41], 12, 14 * 16 // page + 1
    ents = len(starts)
    pages = ents * cols
    table = to_device(r.permutation(pages).reshape(ents, cols).astype(np.int32))
    rope = pa_amd.Rope(nt.freqs(128))
    sc = scales_of(kind)

    def fresh():
        shape = (pages, hkv, page, D)
        pools = [torch.zeros(shape, dtype=torch.float16 if kind == "fp16" else torch.uint8, device="cuda") for _ in range(2)]
        return pools, {**sc, "kv_scales": pa_amd.alloc_kv_scales(pages, hkv, page) if kind == "block" else None}

    def append(c, x, counts, at, positions=None):
        (k, v), kw = c
        return pa_amd.append_rope(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], k, v, table, begins(counts), ints(at), rope,
                                  positions=positions, **kw)

    def read(c, counts, at):
        (k, v), kw = c
        got = pa_amd.read_cache(k, v, table, begins(counts), ints(at), sum(counts), dtype=torch.float32, **kw)
        return [x.double().cpu().numpy() for x in got]

    def tokens(n):
        return torch.from_numpy(r.standard_normal((n, hq + 2 * hkv, D)).astype(np.float16)).cuda()

    cache, plain = fresh(), fresh()
    prompt = tokens(sum(starts))
    for c in (cache, plain):
        append(c, prompt, starts, [0] * ents)
    # Trees: token i at its depth's position, in place start + i.
    parents = [[-1] + [int(r.integers(max(-1, i - 4), i)) for i in range(1, m)] for _ in starts]
    depth = []
    for e, p in enumerate(parents):
        d = []
        for up in p:
            d.append(0 if up < 0 else d[up] + 1)
        depth.append(d)
    pos = ints(s + d for e, s in enumerate(starts) for d in depth[e])
    x = tokens(ents * m)
    q = append(cache, x, [m] * ents, starts, pos)
    rows = pa_amd.tree_rows(parents)
    (k, v), kw = cache
    out = pa_amd.tree_attention(q, k, v, table, begins([m] * ents), ints(starts), rows, **kw)
    K, V = read(cache, [s + m for s in starts], [0] * ents)
    got, qn, at = out.double().cpu().numpy(), q.double().cpu().numpy(), 0
    for e, s in enumerate(starts):
        tree = [int(b) & (2 ** 64 - 1) for b in rows[e * m:(e + 1) * m, 0].tolist()]
        ref, tol = attention(qn[e * m:(e + 1) * m], K[at:at + s + m], V[at:at + s + m], seen_of(s, m, tree), D ** -0.5)
        assert (np.abs(got[e * m:(e + 1) * m] - ref) <= tol).all(), e
        at += s + m
    # The path to each tree's last token is accepted.
    paths = []
    for p in parents:
        path, i = [], m - 1
        while i >= 0:
            path.insert(0, i)
            i = p[i]
        paths.append(path)
    n = [len(p) for p in paths]
    kept = torch.full((ents, m), -9, dtype=torch.int32)
    for e, p in enumerate(paths):
        kept[e, :len(p)] = torch.tensor(p, dtype=torch.int32)
    pa_amd.keep_rows(k, v, table, kept.cuda(), ints(n), ints(starts), kv_scales=kw["kv_scales"])
    took = torch.cat([x[e * m + torch.tensor(p)] for e, p in enumerate(paths)])
    append(plain, took, n, starts)
    a, b = read(cache, [s + c for s, c in zip(starts, n)], [0] * ents), read(plain, [s + c for s, c in zip(starts, n)], [0] * ents)
    for got_rows, want in zip(a, b):
        if kind == "block":   # rounded twice, to scales that may differ: half a step of the larger value each time
            at = 0
            for s, c in zip(starts, n):
                B, lo = drafts.block_of(page), at
                for i in range(s + c):
                    block = slice(lo + i // B * B, min(lo + (i // B + 1) * B, lo + s + c))
                    # A subnormal's step is 2^-9 of the scale, the scale at most 2^-7 of the block's largest.
                    tol = np.abs(want[lo + i]) * 2.0 ** -2 + np.abs(want[block]).max((0, 2))[:, None] * 2.0 ** -13
                    assert (np.abs(got_rows[lo + i] - want[lo + i]) <= tol).all(), (s, i)
                at += s + c
        else:
            np.testing.assert_array_equal(got_rows, want)
    # The next token of each sequence: appended behind the kept rows, decoded.
    lens = [s + c + 1 for s, c in zip(starts, n)]
    q1 = append(cache, tokens(ents), [1] * ents, [s + c for s, c in zip(starts, n)])
    dec = pa_amd.Decoder(hq, hkv, D, page, kind != "fp16", **({"block_scales": True} if kind == "block" else {}))
    dec.plan(torch.tensor(lens, dtype=torch.int32))
    more = {"kv_scales": kw["kv_scales"]} if kind == "block" else {}
    one = dec.run(q1, k, v, table, ints(lens), sc.get("k_scale", 1.0), sc.get("v_scale", 1.0), **more)
    same = pa_amd.tree_attention(q1, k, v, table, begins([1] * ents), ints(s - 1 for s in lens), **kw)
    K, V = read(cache, lens, [0] * ents)
    at = 0
    for e, s in enumerate(lens):
        ref, tol = attention(q1[e:e + 1].double().cpu().numpy(), K[at:at + s], V[at:at + s], np.ones((1, s), bool), D ** -0.5)
        assert (np.abs(same[e].double().cpu().numpy() - ref[0]) <= tol[0]).all(), e
        assert (np.abs(one[e].double().cpu().numpy() - ref[0]) <= 2e-3 * np.abs(V[at:at + s]).max()).all(), e
        at += s


@pytest.mark.parametrize("kind", ["fp16", "block"])
def test_caches_past_32_bits(kind):
    """Pages whose bytes lie past 4 GiB: attention, rows kept, rows read."""
    hkv, page = 8, 16
    small = Cache(kind, page, hkv, 2, 6, seed=5)
    pages = (9 if kind == "fp16" else 5) * 2 ** 30 // (hkv * page * D * (2 if kind == "fp16" else 1))
    shift = pages - small.pages            # the small cache's pages are the large one's last
    dt = torch.float16 if kind == "fp16" else torch.uint8
    pools = []
    for x in small.kv:
        t = torch.empty((pages, hkv, page, D), dtype=dt, device="cuda")
        t[shift:] = torch.from_numpy(x).cuda()
        pools.append(t)
    scales = None
    if kind == "block":
        scales = pa_amd.alloc_kv_scales(pages, hkv, page)
        scales.view(pages, -1)[shift:] = torch.from_numpy(small.scales).cuda().view(small.pages, -1)
    table = torch.from_numpy(small.table + shift).cuda()
    entries, r = [(60, 9), (3, 40)], np.random.default_rng(1)
    n = sum(m for _, m in entries)
    q = r.standard_normal((n, 16, D)).astype(np.float16)
    trees = [random_tree(r, m) for _, m in entries]
    tb, starts = begins([m for _, m in entries]), ints(s for s, _ in entries)
    out = pa_amd.tree_attention(torch.from_numpy(q).cuda(), *pools, table, tb, starts,
                                drafts.tree_bits([b for t in trees for b in t], 1), kv_scales=scales)
    check_attention(small, entries, 16, trees, out, q)
    pa_amd.keep_rows(*pools, table, ints([2, 4, 5, 0, 7, 30]).view(2, 3), ints([3, 3]), starts, kv_scales=scales)
    drafts.keep(small, [(0, 60, [2, 4, 5]), (1, 3, [0, 7, 30])])
    for got, want in zip(pools, small.kv):
        np.testing.assert_array_equal(got[shift:].cpu().numpy().view(np.uint8), want.view(np.uint8))
    got = pa_amd.read_cache(*pools, table, begins([69, 43]), ints([0, 0]), 112, dtype=torch.float32, kv_scales=scales)
    for j in range(2):
        want = np.concatenate([small.rows(j, 0, 0, 69), small.rows(j, 1, 0, 43)])
        np.testing.assert_array_equal(got[j].double().cpu().numpy(), want)


def test_rows_past_32_bits():
    """Token strides of 2^25 elements."""
    cache, n, hq = Cache("fp16", 16, 2, 1, 10, seed=5), 80, 4
    r = np.random.default_rng(3)
    q = r.standard_normal((n, hq, D)).astype(np.float16)
    far = torch.empty(79 * 2 ** 25 + hq * D, dtype=torch.float16, device="cuda").as_strided((n, hq, D), (2 ** 25, D, 1))
    far.copy_(torch.from_numpy(q))
    k, v, table, _ = cache.device()
    pa_amd.tree_attention(far, k, v, table, begins([n]), ints([50]), out=far)
    check_attention(cache, [(50, n)], hq, None, far.contiguous(), q)
    big = far[:, :2]
    pa_amd.read_cache(k, v, table, begins([n]), ints([50]), n, k_out=big)
    np.testing.assert_array_equal(big.double().cpu().numpy(), cache.rows(0, 0, 50, 50 + n))


@pytest.mark.parametrize("kind,page", [("fp16", 5000), ("fp8", 4004), ("block", 4008), ("fp16", 4999)])
def test_large_pages(kind, page):
    entries = [(page + 17, 20), (page - 4, 9)]
    cache = Cache(kind, page, 1, 2, 2, seed=page)
    trees = [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    out, q = run_attention(cache, entries, 4, trees)
    check_attention(cache, entries, 4, trees, out, q)


def test_graphs_that_share_memory():
    """Two captured calls out of one pool of memory, replayed in turn with eager calls between them."""
    cache = Cache("fp16", 16, 2, 2, 40, seed=3)
    k, v, table, _ = cache.device()
    r = np.random.default_rng(2)
    q = [torch.from_numpy(r.standard_normal((n, 8, D)).astype(np.float16)).cuda() for n in (9, 70)]
    starts = [ints([500]), ints([510])]
    outs = [torch.empty_like(x) for x in q]
    want = [pa_amd.tree_attention(x, k, v, table, begins([x.size(0)]), s) for x, s in zip(q, starts)]
    tb = [begins([x.size(0)]) for x in q]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in q]
    pool = None
    for g, x, s, t, o in zip(graphs, q, starts, tb, outs):
        with torch.cuda.graph(g, pool=pool):
            pa_amd.tree_attention(x, k, v, table, t, s, out=o)
        pool = g.pool()
    for _ in range(4):
        for g, o, w, x, s, t in zip(graphs, outs, want, q, starts, tb):
            o.fill_(5.0)
            g.replay()
            assert torch.equal(pa_amd.tree_attention(x, k, v, table, t, s), w)
            torch.cuda.synchronize()
            assert torch.equal(o, w)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
def test_scales(kind, scale):
    """No scale: the mean of what is seen; a negative one; one that leaves few places."""
    cache = Cache(kind, 16, 2, 2, 6, seed=9)
    entries = [(50, 9), (0, 30)]
    trees = [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    out, q = run_attention(cache, entries, 8, trees, sm_scale=scale)
    check_attention(cache, entries, 8, trees, out, q, scale=scale)


def test_one_query_for_all_and_one_that_is_not_a_number():
    cache, n = Cache("fp16", 16, 2, 1, 8, seed=9), 40
    k, v, table, _ = cache.device()
    r = np.random.default_rng(4)
    row = r.standard_normal((1, 8, D)).astype(np.float16)
    out = pa_amd.tree_attention(torch.from_numpy(row).cuda().expand(n, 8, D), k, v, table, begins([n]), ints([66]))
    check_attention(cache, [(66, n)], 8, None, out, np.repeat(row, n, 0))
    q = np.repeat(row, n, 0)
    q[11, 3, 5], q[12, 0, 0] = np.nan, np.inf
    bad = pa_amd.tree_attention(torch.from_numpy(q).cuda(), k, v, table, begins([n]), ints([66]))
    assert bad[11, 3].isnan().all() and bad[12, 0].isnan().all()
    bad[11, 3], bad[12, 0] = out[11, 3], out[12, 0]
    assert torch.equal(bad, out)


@pytest.mark.parametrize("chain", [False, True])
def test_values_past_fp16_in_block_scales(chain):
    """A code and scale that no append writes, 448 * 2^8: infinite for the tokens that see it, nothing to the others."""
    cache, start, n = Cache("block", 16, 2, 1, 4, seed=8), 32, 12
    page = cache.table[0, start // 16]
    cache.scales[page, :, 0, 1] = 135
    cache.kv[1][page] = 0x38                       # ones, 256 with the scale
    cache.kv[1][page, :, 7, 3], cache.kv[1][page, :, 7, 90] = 0x7e, 0xfe
    tree = [(1 << i) | (1 << 7 if i == 9 else 0) for i in range(n)]
    out, _ = run_attention(cache, [(start, n)], 8, None if chain else [tree])
    see = seen_of(start, n, None if chain else tree)[:, start + 7]
    got = out.float().cpu().numpy()
    assert (got[see][:, :, 3] == np.inf).all() and (got[see][:, :, 90] == -np.inf).all() and see.any() and not see.all()
    got[np.ix_(see, range(8), [3, 90])] = 0
    assert np.isfinite(got).all()


def test_no_tokens():
    cache = Cache("block", 16, 2, 2, 4, seed=9)
    k, v, table, scales = cache.device()
    q = torch.empty((0, 8, D), dtype=torch.float16, device="cuda")
    none = ints([0, 0, 0])
    assert pa_amd.tree_attention(q, k, v, table, none, ints([3, 4]), kv_scales=scales).shape == (0, 8, D)
    assert [x.shape for x in pa_amd.read_cache(k, v, table, none, ints([3, 4]), 0, kv_scales=scales)] == [(0, 2, D)] * 2
    pa_amd.keep_rows(k, v, table, torch.empty((2, 0), dtype=torch.int32, device="cuda"), ints([0, 0]), ints([3, 4]), kv_scales=scales)
    # Entries without tokens among ones that have some, tokens that no entry holds: left as they were.
    out = torch.full((6, 8, D), 3.0, dtype=torch.float16, device="cuda")
    q = torch.ones_like(out)
    pa_amd.tree_attention(q, k, v, table, ints([2, 2, 2]), ints([3, 4]), kv_scales=scales, out=out)
    pa_amd.keep_rows(k, v, table, ints([4, 5, 6, 7]).view(2, 2), ints([0, -3]), ints([3, 4]), kv_scales=scales)
    assert (out == 3).all()
    for got, want in zip((k, v), cache.kv):
        np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["fp16", "fp8"])
def test_one_token_of_a_long_sequence(kind):
    start = 300_001
    cache = Cache(kind, 128, 1, 1, cols_for([(start, 1)], 128), seed=3)
    out, q = run_attention(cache, [(start, 1)], 2, None)
    check_attention(cache, [(start, 1)], 2, None, out, q)
