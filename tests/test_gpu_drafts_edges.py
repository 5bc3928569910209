"""GPU tests of the drafted-token operators at the edges of what they take: places up to 2^31 - 258, tree rows with fewer
or more bits than tokens, more accepted rows than a list holds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import drafts
import pa_amd
from drafts import D, Cache, random_tree
from test_gpu_drafts import begins, check_attention, cols_for, ints, run_attention

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]

LAST = 2 ** 31 - 257      # an entry's places end here at most


def test_the_last_places():
    """A sequence of 2^31 - 257 places, every entry of its table but the last one page of 2^16 tokens: the softmax is that over
    its rows, 2^15 - 1 times each, and the last page's, one of whose places weighs as much as all others. The entry beside,
    one place longer, is left out."""
    page, n, hq = 2 ** 16, 3, 2
    cache = Cache("fp8", page, 1, 1, 2, seed=3, spare=0)
    sign = np.where(np.random.default_rng(0).random(D) < 0.5, -1.0, 1.0)
    own, slot = int(cache.table[0, 1]), LAST % page - 9
    cache.kv[0][own, 0, slot] = np.where(sign > 0, 0x6c, 0xec)      # 96 * 0.02: a score of 21.7, ln 2^31 is 21.5
    k, v, _, _ = cache.device()
    table = torch.full((1, 2 ** 15), int(cache.table[0, 0]), dtype=torch.int32, device="cuda")
    table[0, -1] = own
    q = np.tile(sign, (2 * n, hq, 1)).astype(np.float16)
    out = torch.full((2 * n, hq, D), 5.0, dtype=torch.float16, device="cuda")
    pa_amd.tree_attention(torch.from_numpy(q).cuda(), k, v, table, begins([n, n]), ints([LAST - n, LAST - n + 1]), None, out=out,
                          slot_ids=ints([0, 0]), **cache.kw(None))
    got = out.double().cpu().numpy()
    assert (got[n:] == 5).all()
    K, V = (cache.rows(j, 0, 0, 2 * page)[:, 0] for j in range(2))
    s = K @ sign / D ** 0.5
    for i in range(n):
        seen = (LAST - n + i) % page + 1                    # of the last page
        times = np.concatenate([np.full(page, 2.0 ** 15 - 1), np.arange(page) < seen])
        p = np.exp(s - s[page + slot]) * times
        assert 0.2 < p[page + slot] / p.sum() < 0.8
        p /= p.sum()
        size = p @ np.abs(V)
        # attention()'s tolerance, sums in runs of at most 2^31 / 256 blocks / 8 (a lane has every fourth place of a
        # stream, a sum of the products 16 at once).
        err = drafts.SCORE_REL / D ** 0.5 * np.abs(K).sum(1).max()
        tol = size * (2.0 ** -11 + 2 * err + 2.0 ** 20 * 2.0 ** -24) + np.abs(p @ V) * 2.0 ** -11 + 2.0 ** -24
        for h in range(hq):
            assert (np.abs(got[i, h] - p @ V) <= tol).all(), (i, h, np.abs(got[i, h] - p @ V).max())


def test_values_that_are_not_finite_at_the_last_places():
    """The same table: one that all tokens see, one that the second token brings."""
    page, n, hq = 2 ** 16, 3, 2
    cache = Cache("fp8", page, 1, 1, 2, seed=3, spare=0)
    own = int(cache.table[0, 1])
    cache.kv[1][own, 0, LAST % page - 9, 5] = 0x7f
    cache.kv[1][own, 0, LAST % page - 2, 9] = 0xff
    k, v, _, _ = cache.device()
    table = torch.full((1, 2 ** 15), int(cache.table[0, 0]), dtype=torch.int32, device="cuda")
    table[0, -1] = own
    q = torch.randn((n, hq, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    got = pa_amd.tree_attention(q, k, v, table, begins([n]), ints([LAST - n]), **cache.kw(None)).cpu().numpy()
    want = np.zeros((n, hq, D), bool)
    want[:, :, 5] = want[1:, :, 9] = True
    np.testing.assert_array_equal(np.isnan(got), want)
    assert np.isfinite(got[~want]).all()


@pytest.mark.parametrize("kind", ["fp16", "block"])
def test_rows_at_the_last_places(kind):
    """Rows read and kept at the end of 2^31 places."""
    page, n = 2 ** 16, 40
    cache = Cache(kind, page, 2, 1, 1, seed=4, spare=0)
    k, v, _, scales = cache.device()
    table = torch.zeros((1, 2 ** 15), dtype=torch.int32, device="cuda")
    at = 2 ** 31 - 128
    got = pa_amd.read_cache(k, v, table, begins([n]), ints([at]), n, dtype=torch.float32, kv_scales=scales)
    for j in range(2):
        np.testing.assert_array_equal(got[j].double().cpu().numpy(), cache.rows(j, 0, at % page, at % page + n))
    pa_amd.keep_rows(k, v, table, ints([0, 3, 9, 21]).view(1, 4), ints([4]), ints([at]), kv_scales=scales)
    drafts.keep(cache, [(0, at % page, [0, 3, 9, 21])])
    for x, want in zip((k, v), cache.kv):
        np.testing.assert_array_equal(x.cpu().numpy().view(np.uint8), want.view(np.uint8))
    # Read past the end: the last places, then none.
    out = torch.full((n, 2, D), 7.0, dtype=torch.float32, device="cuda")
    pa_amd.read_cache(k, v, table, begins([n]), ints([2 ** 31 - 5]), n, dtype=torch.float32, k_out=out, kv_scales=scales)
    np.testing.assert_array_equal(out[:5].double().cpu().numpy(), cache.rows(0, 0, page - 5, page))
    assert (out[5:] == 7).all()


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("start", [2 ** 31 - 10, 2 ** 31 - 36])
def test_rows_kept_to_the_last_place(kind, start):
    """The last places of all, and numbers that would lie behind them."""
    page = 2 ** 16
    cache = Cache(kind, page, 2, 1, 1, seed=4, spare=0)
    k, v, _, scales = cache.device()
    table = torch.zeros((1, 2 ** 15), dtype=torch.int32, device="cuda")
    pa_amd.keep_rows(k, v, table, ints([1, 3, 9, 12, 30, 40, 2 ** 31 - 1]).view(1, 7), ints([7]), ints([start]), kv_scales=scales)
    here = start % page
    drafts.keep(cache, [(0, here, [j for j in (1, 3, 9, 12, 30) if here + j < page])])
    for x, want in zip((k, v), cache.kv):
        np.testing.assert_array_equal(x.cpu().numpy().view(np.uint8), want.view(np.uint8))
    if scales is not None:
        np.testing.assert_array_equal(scales.cpu().numpy(), cache.scales)


@pytest.mark.parametrize("n,words", [(100, 1), (129, 2), (3, 5), (64, 1), (64, 3), (200, 4)])
def test_tree_rows_with_fewer_or_more_bits(n, words):
    """Tokens past a row's bits are not seen; bits past the entry's tokens name none."""
    r = np.random.default_rng(n)
    entries = [(50, n), (3, min(n, 40))]
    cache = Cache("fp16", 16, 2, 2, cols_for(entries, 16), seed=n)
    full = [random_tree(r, m, spread=60) for _, m in entries]
    given = [[x | int(r.integers(0, 2)) << (64 * words - 1) if m <= 64 * words - 1 else x for x in t]
             for t, (_, m) in zip(full, entries)]
    out, q = run_attention(cache, entries, 4, given, words=words)
    seen = [[x & (2 ** (64 * words) - 1) for x in t] for t in full]
    check_attention(cache, entries, 4, seen, out, q)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
def test_more_kept_rows_than_the_list_holds(kind):
    cache = Cache(kind, 16, 2, 3, 4, seed=6)
    k, v, table, scales = cache.device()
    kept = [[1, 2, 5], [0, 4, 6], [2, 3, 4]]
    pa_amd.keep_rows(k, v, table, ints(sum(kept, [])).view(3, 3), ints([7, 2 ** 31 - 1, -2 ** 31]), ints([10, 20, 30]), kv_scales=scales)
    drafts.keep(cache, [(0, 10, kept[0]), (1, 20, kept[1]), (2, 30, [])])
    for x, want in zip((k, v), cache.kv):
        np.testing.assert_array_equal(x.cpu().numpy().view(np.uint8), want.view(np.uint8))


def test_no_entry_has_the_tokens():
    """Every entry out of range: nothing is written, and the next call over the same memory is right."""
    entries = [(30, 4), (9, 3)]
    cache = Cache("fp16", 16, 2, 2, cols_for(entries, 16), seed=2)
    k, v, table, _ = cache.device()
    q = torch.randn((7, 4, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).half()
    out = torch.full_like(q, 3.0)
    for starts, slots in (([-1, -2 ** 31], [0, 1]), ([30, 9], [2, -1]), ([2 ** 31 - 1, 2 ** 31 - 2], [0, 1])):
        pa_amd.tree_attention(q, k, v, table, begins([4, 3]), ints(starts), None, slot_ids=ints(slots), out=out)
        assert (out == 3).all()
    pa_amd.tree_attention(q, k, v, table, begins([4, 3]), ints([30, 9]), None, out=out)
    check_attention(cache, entries, 4, None, out, q.cpu().numpy())
