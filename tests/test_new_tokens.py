"""CPU tests of the new-token operators: what their C entry points refuse before anything is launched, block sizes,
and the tests' own plain model of a block-scaled cache."""

import ctypes

import numpy as np
import pytest

import new_tokens as nt
import oracle
import pa_amd
from pa_amd import _lib

BAD, LONG = _lib.PA_ERR_INVALID_ARGUMENT, _lib.PA_ERR_LENGTH
A = 1 << 20   # an address that nothing reads: every call here is refused first


def rows(heads=8, stride=None, out=A + (1 << 19), **kw):
    r = _lib.HeadRows()
    r.in_, r.heads, r.eps = A, heads, 1e-6
    r.in_stride = r.out_stride = heads * 128 if stride is None else stride
    r.out = out
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def norm(q=None, k=None, positions=A, n=4, rope=None):
    ref = lambda r: None if r is None else ctypes.byref(r)   # noqa: E731
    return _lib.load().pa_norm_rope(rope, ref(q), ref(k), positions, n, None)


def message() -> str:
    return _lib.load().pa_last_error().decode()


def test_block_tokens():
    assert [pa_amd.block_tokens(p) for p in (8, 16, 24, 32, 40, 48, 128)] == [8, 16, 8, 16, 8, 16, 16]
    assert all(pa_amd.block_tokens(p) == 0 for p in (0, -8, 1, 4, 12, 100))
    assert pa_amd.kv_dtype_name(pa_amd.FP8_E4M3_BLOCK) == "fp8_e4m3_block"
    assert pa_amd.kv_dtype_bytes(pa_amd.FP8_E4M3_BLOCK) == 1
    assert pa_amd.tile_tokens(pa_amd.FP8_E4M3_BLOCK, 128, 4) == pa_amd.tile_tokens(pa_amd.FP8_E4M3, 128, 4)


def test_bytes_per_page_counts_the_scales():
    cfg = pa_amd.CacheConfig(4, 16, 8, 128, 4, 4, pa_amd.FP8_E4M3_BLOCK, 1.0, 1.0)
    assert pa_amd.PagedKVCache.bytes_per_page(cfg) == 2 * 8 * 16 * 128 + 2 * 8
    cfg.page_size = 24
    assert pa_amd.PagedKVCache.bytes_per_page(cfg) == 2 * 8 * 24 * 128 + 2 * 8 * 3


@pytest.mark.parametrize("change,word", [
    (dict(in_=None), "null rows"), (dict(in_=A + 8), "aligned"), (dict(in_stride=1028), "aligned"),
    (dict(in_stride=-1024), "aligned"), (dict(in_stride=2**26), "aligned"), (dict(out_stride=-1024), "aligned"),
    (dict(out=None), "null output"), (dict(out=A + (1 << 19) + 4), "aligned"), (dict(out_stride=1020), "aligned"),
    (dict(out_stride=512), "rows overlap"), (dict(out_stride=0), "rows overlap"),
    (dict(weight=A + 4), "weight"), (dict(weight=A, eps=-1.0), "eps"), (dict(weight=A, eps=float("nan")), "eps"),
    (dict(weight=A, eps=1e-39), "eps"),
    (dict(heads=-1), "negative"), (dict(out=A + 1024), "overlaps"), (dict(out=A - 2048), "overlaps"),
    (dict(out=A, out_stride=2048), "overlaps"),
])
def test_norm_rope_refuses_rows(change, word):
    for q, k in ((rows(**change), None), (None, rows(**change)), (rows(), rows(**change))):
        assert norm(q, k) == BAD and word in message(), message()


def test_norm_rope_refuses_sizes():
    assert norm(rows(), n=-1) == BAD
    assert norm(rows(), n=2**31 // (16 * 8)) == LONG and "INT_MAX" in message()
    assert norm(n=5) == _lib.PA_OK and norm(rows(), n=0) == _lib.PA_OK    # nothing to do: no launch


@pytest.mark.parametrize("args,word", [
    ((8,), "rot_dim"), ((136,), "rot_dim"), ((24,), "rot_dim"), ((0,), "rot_dim"),
    ((64, 0), "axes"), ((64, 5), "axes"), ((64, 2), "axis"),
])
def test_rope_refuses_shapes(args, word):
    f = np.ones(64)
    h = ctypes.c_void_p()
    rot, axes = args[0], args[1] if len(args) > 1 else 1
    assert _lib.load().pa_rope_create(f.ctypes.data, None, rot, axes, 0, 1.0, ctypes.byref(h)) == BAD
    assert word in message() and not h.value


def test_rope_refuses_values():
    lib, h = _lib.load(), ctypes.c_void_p()
    f, a = np.ones(64), np.zeros(64, np.int32)
    for bad in (np.nan, np.inf):
        f[31] = bad
        assert lib.pa_rope_create(f.ctypes.data, None, 64, 1, 0, 1.0, ctypes.byref(h)) == BAD and "finite" in message()
    f[31] = 1.0
    assert lib.pa_rope_create(f.ctypes.data, None, 64, 1, 0, np.inf, ctypes.byref(h)) == BAD
    for bad in (-1, 2):
        a[5] = bad
        assert lib.pa_rope_create(f.ctypes.data, a.ctypes.data, 64, 2, 0, 1.0, ctypes.byref(h)) == BAD
    assert lib.pa_rope_create(None, None, 64, 1, 0, 1.0, ctypes.byref(h)) == BAD
    assert lib.pa_rope_dim(None) == 0 and lib.pa_rope_axes(None) == 0
    lib.pa_rope_destroy(None)
    with pytest.raises(pa_amd.InvalidArgument):
        pa_amd.Rope(np.ones((2, 32)))
    with pytest.raises(pa_amd.InvalidArgument):
        pa_amd.Rope(np.ones(32), axes=np.zeros(16))


def append(dtype=pa_amd.FP8_E4M3_BLOCK, q=None, k=None, **kw):
    a = _lib.AppendArgs()
    a.num_tokens, a.num_entries, a.tok_begin, a.start_pos = 4, 2, A, A
    a.v, a.v_stride, a.k_cache, a.v_cache, a.kv_scales = A, 1024, A, A, A
    a.block_table, a.block_table_stride, a.num_table_rows, a.num_pages = A, 4, 2, 8
    a.page_size, a.k_scale, a.v_scale = 16, 1.0, 1.0
    for name, v in kw.items():
        setattr(a, name, v)
    k = rows() if k is None else k
    return _lib.load().pa_append_rope(dtype, ctypes.byref(a), None, None if q is None else ctypes.byref(q),
                                      ctypes.byref(k), None)


@pytest.mark.parametrize("change,word", [
    (dict(num_tokens=-1), "sizes"), (dict(num_entries=-1), "sizes"), (dict(page_size=0), "sizes"),
    (dict(block_table_stride=0), "sizes"), (dict(num_table_rows=-1), "sizes"), (dict(num_pages=-1), "sizes"),
    (dict(v=None), "v is null"), (dict(v=A + 2), "aligned"), (dict(v_stride=100), "aligned"), (dict(v_stride=-1024), "aligned"),
    (dict(tok_begin=None), "null"), (dict(start_pos=None), "null"), (dict(block_table=None), "null"),
    (dict(k_cache=None), "null"), (dict(v_cache=None), "null"), (dict(k_cache=A + 8), "caches"),
    (dict(kv_scales=None), "kv_scales"), (dict(kv_scales=A + 1), "kv_scales"),
    (dict(page_size=12), "multiple of 8"), (dict(page_size=4), "multiple of 8"),
])
def test_append_rope_refuses(change, word):
    assert append(**change) == BAD and word in message(), message()


def test_append_rope_refuses_rows_and_types():
    assert append(dtype=7) == BAD and append(k=rows(heads=0)) == BAD
    assert append(k=rows(in_=A + 2)) == BAD and append(q=rows(out=None)) == BAD
    assert append(num_tokens=2**31 // (16 * 24)) == LONG
    assert append(num_tokens=0) == _lib.PA_OK and append(num_entries=0) == BAD
    for bad in (dict(k_scale=0.0), dict(v_scale=float("nan")), dict(k_scale=float("inf"))):
        assert append(dtype=pa_amd.FP8_E4M3, **bad) == BAD and "scale" in message()
    lib, k = _lib.load(), rows()
    assert lib.pa_append_rope(0, None, None, None, ctypes.byref(k), None) == BAD
    assert lib.pa_cache_append_rope(None, None, None, 0, None, None, None, ctypes.byref(k), A, 1024, None, None) == BAD
    # The per-tensor append does not write block-scaled caches.
    assert lib.pa_append_quantize(2, A, A, A, A, A, 0, 4, 8, 128, 16, 1.0, 1.0, None) == BAD
    assert "pa_append_rope" in message()


def test_decode_refuses_block_scales():
    p = _lib.DecodeParams()
    p.num_q_heads, p.num_kv_heads, p.head_dim, p.num_ctas, p.page_size, p.batch = 32, 8, 128, 4, 16, 1
    p.block_table_stride = 1
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "segments", "cta_seg_begin", "item_seg_begin"):
        setattr(p, f, A)
    for scales in (None, A + 2):
        p.kv_scales = scales
        with pytest.raises(pa_amd.InvalidArgument, match="kv_scales"):
            pa_amd.decode_split(pa_amd.FP8_E4M3_BLOCK, p, 0)
    p.kv_scales, p.page_size = A, 20
    with pytest.raises(pa_amd.InvalidArgument, match="multiple of 8"):
        pa_amd.decode_split(pa_amd.FP8_E4M3_BLOCK, p, 0)
    with pytest.raises(RuntimeError, match="block_scales"):
        pa_amd.Decoder(32, 8, 128, 16, False, block_scales=True)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        pa_amd.Decoder(32, 8, 128, 20, True, block_scales=True)


def test_cache_refuses_block_configs():
    h = ctypes.c_void_p()
    for page, ks in ((20, 1.0), (16, 0.5)):
        cfg = pa_amd.CacheConfig(4, page, 8, 128, 4, 4, pa_amd.FP8_E4M3_BLOCK, ks, 1.0)
        assert _lib.load().pa_cache_create(ctypes.byref(cfg), ctypes.byref(h)) == BAD


def test_plain_e4m3_is_the_oracles():
    x = np.concatenate([np.linspace(-500, 500, 4001), 2.0 ** np.linspace(-14, 9, 2001), -2.0 ** np.arange(-12, 9.0),
                        [0.0, -0.0, np.inf, -np.inf, 448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10]]).astype(np.float32)
    assert np.array_equal(nt.e4m3_encode(x), oracle.f32_to_e4m3(x))


def test_plain_block_pool():
    """A block that grows in steps holds every value within half a step of its type, under the scale its largest
    value asks for, whatever the steps."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 2, 128)) * 2.0 ** rng.integers(-3, 4, (40, 1, 1))
    table = [2, 0, 1]
    for steps in ([40], [1] * 40, [7, 16, 17]):
        pool = nt.BlockPool(np.zeros((3, 2, 16, 128), np.uint8), np.full((3, 2, 1), 127))
        at = 0
        for n in steps:
            pool.append(x[at:at + n], at, table)
            at += n
        for t in range(40):
            got = pool.values()[table[t // 16], :, t % 16]
            for h in range(2):
                top = np.abs(x[t // 16 * 16:t // 16 * 16 + 16, h]).max()
                k = pool.exps[table[t // 16], h, 0]
                assert k == nt.exponent(top) and 224 * 2.0 ** k < top <= 448 * 2.0 ** k
                # Rounded twice where the scale grew: half a step of the values, and half of the last grid.
                tol = np.maximum(np.abs(x[t, h]) * 2.0 ** -4, 2.0 ** (k - 10)) + 2.0 ** (k - 10)
                assert np.all(np.abs(got[h] - x[t, h]) <= tol)
