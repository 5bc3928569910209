"""CPU tests of the drafted-token operators: what their C entry points refuse before anything is launched, calls with
nothing to do, tree_rows, and the tests' own plain model of keeping rows."""

import ctypes

import numpy as np
import pytest
import torch

import drafts
import pa_amd
from pa_amd import _lib
from test_new_tokens import A, BAD, LONG, message, rows

BLOCK = pa_amd.FP8_E4M3_BLOCK


def cached(**kw):
    c = _lib.CachedTokens()
    c.num_tokens, c.num_entries, c.tok_begin, c.start_pos = 4, 2, A, A
    c.k_cache, c.v_cache, c.kv_scales, c.block_table = A, A, A, A
    c.block_table_stride, c.num_table_rows, c.num_pages, c.page_size, c.num_kv_heads = 4, 2, 8, 16, 8
    c.k_scale = c.v_scale = 1.0
    for name, v in kw.items():
        setattr(c, name, v)
    return c


def attend(dtype=BLOCK, q=None, tree=None, words=0, scale=0.1, ws=None, ws_bytes=0, **kw):
    c, q = cached(**kw), rows() if q is None else q
    return _lib.load().pa_tree_attention(dtype, ctypes.byref(c), ctypes.byref(q), tree, words, scale, ws, ws_bytes, None)


def read(dtype=BLOCK, type=0, k=A, ks=1024, v=A + (1 << 19), vs=1024, **kw):
    c = cached(**kw)
    return _lib.load().pa_read_cache(dtype, ctypes.byref(c), type, k, ks, v, vs, None)


def keep(dtype=BLOCK, kept=A, width=3, counts=A, **kw):
    c = cached(**kw)
    return _lib.load().pa_keep_rows(dtype, ctypes.byref(c), kept, width, counts, None)


SIZES = [
    (dict(num_tokens=-1), "sizes"), (dict(num_entries=-1), "sizes"), (dict(page_size=0), "sizes"),
    (dict(block_table_stride=0), "sizes"), (dict(num_table_rows=-1), "sizes"), (dict(num_pages=-1), "sizes"),
    (dict(num_kv_heads=0), "sizes"), (dict(page_size=12), "multiple of 8"), (dict(page_size=4), "multiple of 8"),
]
POINTERS = [
    (dict(start_pos=None), "null"), (dict(block_table=None), "null"), (dict(k_cache=None), "null"),
    (dict(v_cache=None), "null"), (dict(k_cache=A + 8), "caches"), (dict(v_cache=A + 8), "caches"),
    (dict(kv_scales=None), "kv_scales"), (dict(kv_scales=A + 1), "kv_scales"),
    (dict(k_scale=float("nan")), "finite"), (dict(v_scale=float("inf")), "finite"),
]


@pytest.mark.parametrize("change,word", SIZES + POINTERS)
def test_caches_refused(change, word):
    for call in (attend, read, keep):
        assert call(**change) == BAD and word in message(), (call, message())


def test_long_sizes_refused():
    for call in (attend, read, keep):
        assert call(num_kv_heads=(1 << 14) + 1) == LONG
        assert call(num_entries=(1 << 20) + 1) == LONG
    assert attend(num_tokens=2**31 // (16 * 8)) == LONG
    assert read(num_tokens=2**31 // (16 * 8)) == LONG
    assert keep(num_entries=1 << 20, num_kv_heads=33) == LONG and "2^25" in message()
    assert attend(dtype=7) == BAD and read(dtype=7) == BAD and keep(dtype=-1) == BAD


def test_null_structs_refused():
    lib, q = _lib.load(), rows()
    n = ctypes.c_size_t()
    assert lib.pa_tree_attention(0, None, ctypes.byref(q), None, 0, 1.0, None, 0, None) == BAD
    c = cached()
    assert lib.pa_tree_attention(0, ctypes.byref(c), None, None, 0, 1.0, None, 0, None) == BAD
    assert lib.pa_read_cache(0, None, 0, A, 1024, A, 1024, None) == BAD
    assert lib.pa_keep_rows(0, None, A, 1, A, None) == BAD
    assert lib.pa_tree_attention_workspace(0, None, 8, ctypes.byref(n)) == BAD
    assert lib.pa_tree_attention_workspace(0, ctypes.byref(c), 8, None) == BAD


@pytest.mark.parametrize("q,word", [
    (dict(heads=0), "heads"), (dict(heads=12), "heads"), (dict(heads=8 * 33), "heads"), (dict(heads=-8), "heads"),
    (dict(in_=None), "null"), (dict(in_=A + 8), "aligned"), (dict(in_stride=1028), "aligned"), (dict(out=None), "null"),
    (dict(out_stride=512), "overlap"), (dict(weight=A), "weight"), (dict(out=A + 1024), "overlap"),
])
def test_attention_refuses_rows(q, word):
    assert attend(q=rows(**q)) == BAD and word in message(), message()


def test_attention_refuses_trees_scales_and_entries():
    assert attend(tree=A, words=0) == BAD and "words" in message()
    assert attend(tree=A, words=-1) == BAD and "words" in message()
    assert attend(tree=A + 4, words=1) == BAD and "aligned" in message()
    for bad in (float("nan"), float("inf")):
        assert attend(scale=bad) == BAD and "sm_scale" in message()
    assert attend(dtype=pa_amd.FP8_E4M3, scale=1e38, k_scale=1e5) == BAD and "k_scale must be finite" in message()
    assert attend(tok_begin=None) == BAD and "null" in message()
    assert attend(num_entries=0) == BAD and "no entry" in message()
    assert attend(num_pages=0) == BAD and "pages" in message()
    assert attend(num_tokens=0) == _lib.PA_OK            # nothing to do: no launch
    c, n = cached(num_tokens=0), ctypes.c_size_t(5)
    assert _lib.load().pa_tree_attention_workspace(BLOCK, ctypes.byref(c), 8, ctypes.byref(n)) == _lib.PA_OK and n.value == 0
    assert _lib.load().pa_tree_attention_workspace(BLOCK, ctypes.byref(cached()), 12, ctypes.byref(n)) == BAD


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(type=-1), "type"), (dict(k=A + 8), "aligned"), (dict(v=A + 8), "aligned"),
    (dict(ks=1028), "stride"), (dict(vs=-1024), "stride"), (dict(ks=1 << 26), "stride"), (dict(vs=1016), "overlap"),
    (dict(ks=0), "overlap"), (dict(v=A + 2048), "overlap"), (dict(tok_begin=None), "null"), (dict(num_entries=0), "no entry"),
])
def test_read_refuses(change, word):
    assert read(**change) == BAD and word in message(), message()


def test_read_with_nothing_to_do():
    assert read(num_tokens=0) == _lib.PA_OK and read(k=None, v=None) == _lib.PA_OK
    assert read(num_tokens=0, k=None, v=None, num_entries=0) == _lib.PA_OK
    # Outputs side by side in one buffer do not overlap; their last rows may end where it ends.
    assert read(k=A, ks=2048, v=A + 2048, vs=2048, tok_begin=None) == BAD and "null" in message()
    assert read(k=A, ks=2048, v=A + 2040, vs=2048) == BAD


def test_keep_refuses():
    assert keep(width=-1) == BAD and "width" in message()
    assert keep(kept=None) == BAD and "null" in message()
    assert keep(counts=None) == BAD and "null" in message()
    assert keep(width=0) == _lib.PA_OK and keep(num_entries=0) == _lib.PA_OK


def test_tree_rows():
    rows_ = pa_amd.tree_rows([[-1, 0, 0, 1, 2, -1], [], [-1, -1]], device="cpu")
    assert rows_.dtype == torch.int64 and rows_.tolist() == [[1], [3], [5], [11], [21], [32], [1], [2]]
    chain = pa_amd.tree_rows([[-1] + list(range(129))], device="cpu").numpy().view(np.uint64)
    assert chain.shape == (130, 3)
    for i in range(130):
        assert sum(int(w) << (64 * j) for j, w in enumerate(chain[i])) == (1 << (i + 1)) - 1
    assert pa_amd.tree_rows([], device="cpu").shape == (0, 1)
    for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
        with pytest.raises(pa_amd.InvalidArgument):
            pa_amd.tree_rows([bad], device="cpu")


def test_tensors_refused_without_a_device():
    """The ctypes path's own checks, on CPU tensors."""
    x, t = torch.zeros(2, 4, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(3, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(Exception, match="CUDA"):
        pa_amd.tree_attention(x, pool, pool, t.view(1, 2), t, t[:1])
    with pytest.raises(Exception, match="CUDA"):
        pa_amd.read_cache(pool, pool, t.view(1, 2), t, t[:1], 2)
    with pytest.raises(Exception, match="CUDA"):
        pa_amd.keep_rows(pool, pool, t.view(1, 2), t.view(1, 2), t[:1], t[:1])
    with pytest.raises(RuntimeError, match="dtype"):
        pa_amd.read_cache(pool, pool, t.view(1, 2), t, t[:1], 2, dtype=torch.float64)


def test_plain_keep():
    """The model itself: rows move to the front in order, blocks that gain a row take the scale of what they keep."""
    c = drafts.Cache("fp16", 8, 1, 1, 4, seed=1)
    before = c.rows(0, 0, 0, 32)
    drafts.keep(c, [(0, 10, [0, 3, 4])])
    want = before.copy()
    want[11], want[12] = before[13], before[14]
    np.testing.assert_array_equal(c.rows(0, 0, 0, 32), want)
    b = drafts.Cache("block", 8, 1, 1, 4, seed=1)
    before, scales = b.rows(0, 0, 0, 32), b.scales.copy()
    drafts.keep(b, [(0, 8, [1, 9])])
    page = b.table[0, 1]
    assert (np.abs(b.rows(0, 0, 8, 10) - before[[9, 17]]) <= np.abs(before[[9, 17]]) * 2.0 ** -4).all()
    k = int(b.scales[page, 0, 0, 0]) - 127
    assert 224 * 2.0 ** k < np.abs(before[[9, 17]]).max() <= 448 * 2.0 ** k
    others = [p for p in range(b.pages) if p != page]
    np.testing.assert_array_equal(b.scales[others], scales[others])


def test_plain_attention():
    """The model against sums written out, and a row that sees nothing."""
    r = np.random.default_rng(0)
    q, k, v = r.standard_normal((2, 2, 128)), r.standard_normal((3, 1, 128)), r.standard_normal((3, 1, 128))
    out, _ = drafts.attention(q, k, v, np.array([[1, 0, 1], [0, 0, 0]], bool), 0.3)
    e = [np.exp(0.3 * (q[0, 1] @ k[j, 0])) for j in (0, 2)]
    np.testing.assert_allclose(out[0, 1], (e[0] * v[0, 0] + e[1] * v[2, 0]) / sum(e), rtol=1e-12)
    assert (out[1] == 0).all()
