"""Drafted tokens over a paged cache on the device, against plain forms in 64 bits: attention of several tokens per
sequence, accepted rows kept, rows read back."""

import numpy as np
import pytest
import torch

import drafts
import pa_amd
from drafts import D, Cache, attention, random_tree, seen_of

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32).cuda()


def begins(counts, first=0):
    return ints(np.concatenate([[first], first + np.cumsum(counts)]))


def cols_for(entries, page):
    return max(-(-(s + n) // page) for s, n in entries) if entries else 1


def run_attention(cache, entries, hq, trees, seed=1, words=None, q=None, **kw):
    """entries: (start, n) of table row e. trees: one list of whole numbers per entry, or None. -> (out, q numpy)"""
    r = np.random.default_rng(seed)
    n = sum(m for _, m in entries)
    if q is None:
        q = (r.standard_normal((n, hq, D)) * 1.5).astype(np.float16)
    k, v, table, scales = cache.device()
    tree = None
    if trees is not None:
        words = words or max([1] + [-(-m // 64) for _, m in entries])
        tree = drafts.tree_bits([row for t in trees for row in t], words)
    out = pa_amd.tree_attention(torch.from_numpy(q).cuda(), k, v, table, begins([m for _, m in entries]),
                                ints(s for s, _ in entries), tree, **cache.kw(scales), **kw)
    return out, q


def check_attention(cache, entries, hq, trees, out, q, scale=None, rows=None):
    out = out.float().cpu().numpy().astype(np.float64)
    at = 0
    for e, (start, n) in enumerate(entries):
        row = e if rows is None else rows[e]
        k, v = (cache.rows(j, row, 0, start + n) for j in range(2))
        ref, tol = attention(q[at:at + n].astype(np.float64), k, v, seen_of(start, n, None if trees is None else trees[e]),
                             1 / np.sqrt(D) if scale is None else scale)
        bad = ~(np.abs(out[at:at + n] - ref) <= tol)
        assert not bad.any(), (f"entry {e} ({start}, {n}): {bad.sum()} off, first at {np.argwhere(bad)[0]}: "
                               f"{out[at:at + n][bad][0]} for {ref[bad][0]} +- {tol[bad][0]}")
        at += n


KINDS = [("fp16", 16), ("fp8", 16), ("block", 16)]


@pytest.mark.parametrize("kind,page", KINDS)
@pytest.mark.parametrize("start,n", [(0, 1), (0, 2), (1, 1), (31, 1), (32, 1), (33, 5), (7, 40), (200, 8), (127, 17), (500, 33)])
@pytest.mark.parametrize("chain", [False, True])
def test_single_sequence(kind, page, start, n, chain):
    cache = Cache(kind, page, 2, 1, cols_for([(start, n)], page), seed=start + n)
    trees = None if chain else [random_tree(np.random.default_rng(n), n)]
    out, q = run_attention(cache, [(start, n)], 8, trees)
    check_attention(cache, [(start, n)], 8, trees, out, q)


@pytest.mark.parametrize("kind,page", [("fp16", 1), ("fp16", 3), ("fp16", 8), ("fp16", 100), ("fp8", 5), ("fp8", 24),
                                       ("fp8", 128), ("block", 8), ("block", 24), ("block", 40), ("block", 64)])
@pytest.mark.parametrize("chain", [False, True])
def test_pages(kind, page, chain):
    entries = [(0, 3), (65, 20), (130, 1), (77, 64), (8, 8)]
    cache = Cache(kind, page, 3, len(entries), cols_for(entries, page), seed=page)
    trees = None if chain else [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    out, q = run_attention(cache, entries, 6, trees)
    check_attention(cache, entries, 6, trees, out, q)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 16, 31, 32])
@pytest.mark.parametrize("n", [1, 9, 70])
def test_groups(group, n):
    entries = [(90, n), (3, max(1, n // 2))]
    cache = Cache("fp16", 16, 2, 2, cols_for(entries, 16), seed=group)
    trees = [random_tree(np.random.default_rng(i), m) for i, (_, m) in enumerate(entries)]
    out, q = run_attention(cache, entries, 2 * group, trees)
    check_attention(cache, entries, 2 * group, trees, out, q)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("n", [63, 64, 65, 130, 200])
def test_wide_trees(kind, n):
    """Rows of several words; n tokens beside an entry of one."""
    entries = [(45, n), (20, 1)]
    cache = Cache(kind, 16, 1, 2, cols_for(entries, 16), seed=n)
    trees = [random_tree(np.random.default_rng(n), m, spread=40) for _, m in entries]
    out, q = run_attention(cache, entries, 4, trees)
    check_attention(cache, entries, 4, trees, out, q)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("start,n,chain", [(3000, 3, False), (4097, 16, False), (2500, 40, False), (2500, 130, True), (700, 300, True)])
def test_long(kind, start, n, chain):
    """Items split over many blocks, and joined."""
    cache = Cache(kind, 16, 2, 1, cols_for([(start, n)], 16), seed=n)
    trees = None if chain else [random_tree(np.random.default_rng(n), n)]
    out, q = run_attention(cache, [(start, n)], 8, trees)
    check_attention(cache, [(start, n)], 8, trees, out, q)


@pytest.mark.parametrize("chain", [False, True])
def test_many_entries(chain):
    """More entries than one look at them takes, some empty, of very different lengths; more items than are split."""
    r = np.random.default_rng(5)
    entries = [(int(r.integers(0, 60)), int(r.integers(0, 4))) for _ in range(700)]
    entries[300] = (900, 7)
    cache = Cache("fp16", 16, 8, 4, 60, seed=2)
    cache.table = r.integers(0, cache.pages, (len(entries), 60)).astype(np.int32)   # pages are shared: only read here
    trees = None if chain else [random_tree(r, n) for _, n in entries]
    out, q = run_attention(cache, entries, 8, trees)
    check_attention(cache, entries, 8, trees, out, q)


def test_rows_that_see_nothing():
    """No earlier place and no bit: zeros; also beside rows that see something."""
    entries = [(0, 5), (40, 3)]
    cache = Cache("fp16", 16, 2, 2, 4)
    trees = [[0, 2, 0, 9, 0], [0, 0, 4]]
    out, q = run_attention(cache, entries, 8, trees)
    check_attention(cache, entries, 8, trees, out, q)
    assert (out[[0, 2, 4]] == 0).all()


@pytest.mark.parametrize("kind", ["fp16", "fp8"])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf", "both"])
@pytest.mark.parametrize("chain", [False, True])
def test_masked_values_do_not_reach(kind, what, chain):
    """Infinities and NaN in the keys and values of tokens that a row does not see leave it as it is; rows that see
    them have them."""
    if kind == "fp8" and "inf" in what:
        pytest.skip("E4M3 has no infinity")
    start, n = 37, 12
    cache = Cache(kind, 16, 2, 1, 4, seed=8)
    vals = {"nan": [np.nan], "inf": [np.inf], "-inf": [-np.inf], "both": [np.inf, -np.inf]}[what]
    for i, x in enumerate(vals):
        page, slot = cache.table[0, (start + 7 + i) // 16], (start + 7 + i) % 16
        cache.kv[1][page, :, slot, 3:90:7] = 0x7f if kind == "fp8" else x
        cache.kv[0][page, :, slot, 5] = 0x7f if kind == "fp8" else np.nan if what == "nan" else cache.kv[0][page, :, slot, 5]
    tree = [(1 << i) | (1 << 7 if i in (9,) else 0) | (1 << 8 if i in (9, 10) else 0) for i in range(n)]
    trees = None if chain else [tree]
    out, q = run_attention(cache, [(start, n)], 8, trees)
    got = out.float().cpu().numpy()
    see = seen_of(start, n, None if chain else tree)
    k, v = (cache.rows(j, 0, 0, start + n) for j in range(2))
    for i in range(n):
        ref, tol = attention(q[i:i + 1].astype(np.float64), k[see[i]], v[see[i]], np.ones((1, see[i].sum()), bool), 1 / np.sqrt(D))
        ok = np.isfinite(ref[0])
        assert (np.abs(got[i][ok] - ref[0][ok]) <= tol[0][ok]).all(), i
        np.testing.assert_array_equal(np.where(np.isnan(got[i]), 0, got[i])[~ok], np.where(np.isnan(ref[0]), 0, ref[0])[~ok])
        np.testing.assert_array_equal(np.isnan(got[i]), np.isnan(ref[0]))


def test_strides_slots_scale_and_padding():
    """q a column of a fused projection, out its own buffer's; table rows by slot_ids; a scale of the caller's;
    tokens of no entry before, behind, and in entries out of range keep what out held."""
    cache = Cache("fp16", 16, 2, 6, 5, seed=4)
    hq, starts, counts = 8, [20, 60, -1, 0, 70], [4, 3, 2, 2, 20]
    rows = [5, 0, 1, 9, 2]                      # the fourth row is out of range, the last entry's places too
    first, n = 2, 2 + sum(counts) + 3
    r = np.random.default_rng(0)
    k, v, table, _ = cache.device()
    fused = torch.from_numpy((r.standard_normal((n, hq + 4, D))).astype(np.float16)).cuda()
    buf = torch.full((n, hq + 1, D), 7.0, dtype=torch.float16, device="cuda")
    q = fused[:, 1:1 + hq]
    got = pa_amd.tree_attention(q, k, v, table, begins(counts, first), ints(starts), None, slot_ids=ints(rows), sm_scale=0.2,
                                out=buf[:, 1:])
    assert got.data_ptr() == buf[:, 1:].data_ptr()
    at = first
    for e in range(2):
        m = counts[e]
        kk, vv = (cache.rows(j, rows[e], 0, starts[e] + m) for j in range(2))
        ref, tol = attention(q[at:at + m].cpu().numpy().astype(np.float64), kk, vv, seen_of(starts[e], m, None), 0.2)
        assert (np.abs(got[at:at + m].float().cpu().numpy() - ref) <= tol).all()
        at += m
    assert (got[:first] == 7).all() and (got[at:] == 7).all() and (buf[:, 0] == 7).all()
    same = q.clone()
    assert torch.equal(pa_amd.tree_attention(same, k, v, table, begins(counts, first), ints(starts), None,
                                             slot_ids=ints(rows), sm_scale=0.2, out=same)[first:at], got[first:at])


def test_bad_pages_read_as_zeros():
    cache = Cache("fp16", 16, 2, 1, 6, seed=4)
    cache.table[0, 1], cache.table[0, 4] = -5, cache.pages
    out, q = run_attention(cache, [(80, 9)], 8, None)
    check_attention(cache, [(80, 9)], 8, None, out, q)


def test_streams_and_graphs():
    """A captured call follows its arrays from replay to replay; calls at once on two streams."""
    entries = [(300, 8), (900, 5)]
    cache = Cache("block", 16, 2, 2, 70, seed=3)
    k, v, table, scales = cache.device()
    r = np.random.default_rng(2)
    q = torch.from_numpy(r.standard_normal((13, 8, D)).astype(np.float16)).cuda()
    tb, starts = begins([8, 5]), ints([300, 900])
    out = torch.empty_like(q)
    args = lambda: dict(kv_scales=scales)
    eager = pa_amd.tree_attention(q, k, v, table, tb, starts, None, **args())
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pa_amd.tree_attention(q, k, v, table, tb, starts, None, out=out, **args())
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(g):
        pa_amd.tree_attention(q, k, v, table, tb, starts, None, out=out, **args())
    for i in range(4):
        starts.copy_(ints([300 - 7 * i, 900 - 111 * i]))
        tb.copy_(ints([0, 8 - i, 13 - i]))
        q.mul_(0.9)
        out.fill_(3.0)
        eager = pa_amd.tree_attention(q, k, v, table, tb, starts, None, out=torch.full_like(q, 3.0), **args())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    want = pa_amd.tree_attention(q, k, v, table, tb, starts, None, out=torch.full_like(q, 3.0), **args())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.full_like(q, 3.0) for _ in streams]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                pa_amd.tree_attention(q, k, v, table, tb, starts, None, out=o, **args())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_repeats_are_equal():
    cache = Cache("fp8", 16, 2, 3, 60, seed=3)
    entries = [(800, 30), (55, 4), (0, 11)]
    trees = [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    first, q = run_attention(cache, entries, 8, trees)
    for _ in range(3):
        assert torch.equal(run_attention(cache, entries, 8, trees, q=q)[0], first)


def test_tree_rows():
    parents = [[-1, 0, 0, 1, 2, -1], [-1] + list(range(69))]
    rows = pa_amd.tree_rows(parents)
    want = [[1, 3, 5, 11, 21, 32], [(1 << (i + 1)) - 1 for i in range(70)]]
    assert torch.equal(rows, drafts.tree_bits([x for w in want for x in w], 2))


def test_ctypes_twin(monkeypatch):
    """The same through ctypes."""
    from pa_amd import ops
    cache = Cache("block", 16, 2, 2, 8, seed=3)
    entries = [(40, 8), (90, 5)]
    trees = [random_tree(np.random.default_rng(i), n) for i, (_, n) in enumerate(entries)]
    a, q = run_attention(cache, entries, 8, trees)
    k, v, table, scales = cache.device()
    read = pa_amd.read_cache(k, v, table, begins([8, 5]), ints([40, 90]), 13, **cache.kw(scales))
    pa_amd.keep_rows(k, v, table, ints([0, 3, 0, 2]).view(2, 2), ints([2, 2]), ints([40, 90]), kv_scales=scales)
    monkeypatch.setattr(ops, "compiled", lambda: None)
    assert torch.equal(run_attention(cache, entries, 8, trees, q=q)[0], a)
    k2, v2, table, scales2 = cache.device()
    again = pa_amd.read_cache(k2, v2, table, begins([8, 5]), ints([40, 90]), 13, **cache.kw(scales2))
    assert all(torch.equal(x, y) for x, y in zip(read, again))
    pa_amd.keep_rows(k2, v2, table, ints([0, 3, 0, 2]).view(2, 2), ints([2, 2]), ints([40, 90]), kv_scales=scales2)
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(scales, scales2)


# ---- reading back

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind,page", [("fp16", 16), ("fp16", 3), ("fp8", 16), ("fp8", 5), ("block", 16), ("block", 24), ("block", 8)])
def test_read_cache(kind, page, dtype):
    cache = Cache(kind, page, 3, 4, 20, seed=page)
    starts, counts = [0, 5, 17, 3], [1, 40, 0, 33]
    counts = [min(c, 20 * page - s) for s, c in zip(starts, counts)]
    k, v, table, scales = cache.device()
    n = sum(counts)
    got = pa_amd.read_cache(k, v, table, begins(counts), ints(starts), n, dtype=dtype, **cache.kw(scales))
    for j in range(2):
        ref = np.concatenate([cache.rows(j, e, s, s + c) for e, (s, c) in enumerate(zip(starts, counts))])
        x = got[j].double().cpu().numpy()
        # One product in 32 bits, then the type's rounding: half a step of each (none where the value is the type's).
        tol = np.abs(ref) * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -20) + (2.0 ** -24 if kind == "fp8" else 0)) + (
            2.0 ** -25 if dtype == torch.float16 else 0)
        assert (np.abs(x - ref) <= tol).all()
        if kind == "block" or (kind == "fp16" and dtype != torch.bfloat16):
            assert torch.equal(got[j].cpu(), torch.from_numpy(ref).to(dtype))


def test_read_cache_leaves_rows():
    """Strided outputs; tokens of no entry and out of range keep what was there."""
    cache = Cache("fp16", 16, 2, 3, 3, seed=1)
    cache.table[1, 1] = cache.pages + 3
    k, v, table, _ = cache.device()
    counts, starts, rows = [3, 20, 2, 5, 4], [45, 10, -1, 0, 2], [0, 1, 2, 7, 2]
    n = 1 + sum(counts) + 2
    buf = torch.full((n, 5, D), 9.0, dtype=torch.float16, device="cuda")
    ko, vo = buf[:, :2], buf[:, 2:4]
    pa_amd.read_cache(k, v, table, begins(counts, 1), ints(starts), n, slot_ids=ints(rows), k_out=ko, v_out=vo)
    want = np.full((n, 5, D), 9.0)
    at = 1
    for e in range(5):
        for i in range(counts[e]):
            pos = starts[e] + i
            if starts[e] >= 0 and rows[e] < 3 and pos < 48 and cache.table[rows[e], pos // 16] < cache.pages:
                for j in range(2):
                    want[at + i, 2 * j:2 * j + 2] = cache.rows(j, rows[e], pos, pos + 1)[0]
        at += counts[e]
    np.testing.assert_array_equal(buf.double().cpu().numpy(), want)


# ---- keeping rows

def check_keep(cache, entries, width, rows=None, more=()):
    k, v, table, scales = cache.device()
    kept = np.full((len(entries), width), 12345678, np.int32)
    for e, (_, ks) in enumerate(entries):
        kept[e, :len(ks)] = ks
    pa_amd.keep_rows(k, v, table, torch.from_numpy(kept).cuda(), ints(len(ks) for _, ks in entries),
                     ints(s for s, _ in entries), kv_scales=scales, slot_ids=None if rows is None else ints(rows))
    drafts.keep(cache, [(e if rows is None else rows[e], s, list(ks)) for e, (s, ks) in enumerate(entries)])
    for got, want in zip((k, v), cache.kv):
        np.testing.assert_array_equal(got.cpu().numpy().view(np.uint8), want.view(np.uint8))
    if scales is not None:
        np.testing.assert_array_equal(scales.cpu().numpy(), cache.scales)


@pytest.mark.parametrize("kind,page", [("fp16", 16), ("fp16", 1), ("fp16", 3), ("fp8", 16), ("fp8", 7), ("block", 8),
                                       ("block", 16), ("block", 24), ("block", 64)])
@pytest.mark.parametrize("seed", range(4))
def test_keep_rows(kind, page, seed):
    r = np.random.default_rng(seed)
    entries = []
    for _ in range(9):
        n = int(r.integers(1, 60))
        entries.append((int(r.integers(0, 50)), sorted(r.choice(n, int(r.integers(0, n + 1)), replace=False).tolist())))
    entries += [(0, [0]), (16, [1]), (15, [0, 1, 2, 3, 4, 40]), (8, list(range(30))), (3, list(range(1, 40)))]
    cache = Cache(kind, page, 3, len(entries), cols_for([(s, 64) for s, _ in entries], page), seed=seed)
    check_keep(cache, entries, 64)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
def test_keep_rows_long(kind):
    r = np.random.default_rng(3)
    entries = [(21, sorted(r.choice(600, 400, replace=False).tolist())), (7, list(range(100)) + list(range(105, 300)))]
    cache = Cache(kind, 16, 2, 2, 45, seed=7)
    check_keep(cache, entries, 400)


@pytest.mark.parametrize("kind", ["fp16", "block"])
def test_keep_rows_out_of_range(kind):
    """Numbers below their index, places past the table, pages and rows out of range: left out."""
    cache = Cache(kind, 16, 2, 3, 4, seed=7)
    cache.table[1, 2] = -1
    entries = [(50, [0, 2, 3, 9, 14, 30, 10 ** 9, 2 ** 31 - 1]), (20, [1, 3, 12, 20, 40]), (5, [2, 3])]
    check_keep(cache, entries, 10, rows=[0, 1, 5])


def test_keep_rows_special_values():
    """NaN codes keep their bytes, zeros ask for the smallest scale, the largest scale stops at 240."""
    cache = Cache("block", 16, 2, 1, 5, seed=7)
    for pos, code in ((20, 0x7f), (21, 0xff), (22, 0x00), (23, 0x80), (33, 0x7e)):
        cache.kv[0][cache.table[0, pos // 16], :, pos % 16] = code
    cache.scales[cache.table[0, 2], 0, 0, 0] = 135
    check_keep(cache, [(18, [2, 3, 4, 5, 15, 16])], 6)
    zero = Cache("block", 16, 2, 1, 5, seed=7)
    for j in range(2):
        zero.kv[j][:] = 0x80
    check_keep(zero, [(16, [1, 2])], 2)


def test_keep_rows_in_a_graph():
    cache = Cache("block", 16, 2, 2, 6, seed=9)
    k, v, table, scales = cache.device()
    kept, counts, starts = ints([1, 3, 5, 0, 2, 9]).view(2, 3), ints([3, 2]), ints([20, 33])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pa_amd.keep_rows(k, v, table, kept, counts, starts, kv_scales=scales)
    for i in range(4):
        counts.copy_(ints([3 - i % 2, 2 + i % 2]))
        starts.copy_(ints([20 + i, 33 - 2 * i]))
        g.replay()
        torch.cuda.synchronize()
        drafts.keep(cache, [(0, 20 + i, [1, 3, 5][:3 - i % 2]), (1, 33 - 2 * i, [0, 2, 9][:2 + i % 2])])
        np.testing.assert_array_equal(k.cpu().numpy(), cache.kv[0])
        np.testing.assert_array_equal(scales.cpu().numpy(), cache.scales)
