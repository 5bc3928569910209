"""CPU tests of the largest sizes that the new-token entry points take: refused before anything is launched."""

from __future__ import annotations

import ctypes

import pytest

from pa_amd import _lib

A = 1 << 40   # an address that nothing reads


def rows(heads, **kw):
    r = _lib.HeadRows()
    r.in_, r.heads, r.in_stride, r.eps = A, heads, 8, 1e-6
    r.out, r.out_stride = A << 2, (1 << 26) - 8
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("heads", [2**19 + 1, 2**23, 2**26])
def test_heads_whose_rows_pass_32_bits(heads):
    """A token of more heads would lie 2^31 bytes and more past its first (2^23), or, in a block, past its first token's
    (15 strides of 2^26 elements before it)."""
    lib, r = _lib.load(), rows(heads)
    one = rows(1)
    for q, k in ((r, None), (None, r), (one, r)):
        ref = [None if x is None else ctypes.byref(x) for x in (q, k)]
        assert lib.pa_norm_rope(None, *ref, None, 1, None) == _lib.PA_ERR_LENGTH and b"heads" in lib.pa_last_error()
    a = _lib.AppendArgs()
    a.num_tokens, a.num_entries, a.tok_begin, a.start_pos = 1, 1, A, A
    a.v, a.v_stride, a.k_cache, a.v_cache, a.kv_scales = A, 8, A, A, A
    a.block_table, a.block_table_stride, a.num_table_rows, a.num_pages = A, 4, 2, 8
    a.page_size, a.k_scale, a.v_scale = 8, 1.0, 1.0
    got = lib.pa_append_rope(2, ctypes.byref(a), None, None, ctypes.byref(r), None)
    assert got == (_lib.PA_ERR_LENGTH if heads < 2**21 else _lib.PA_ERR_INVALID_ARGUMENT)   # (its page passes 2 GiB first)
    got = lib.pa_append_rope(2, ctypes.byref(a), None, ctypes.byref(r), ctypes.byref(one), None)
    assert got == _lib.PA_ERR_LENGTH


def test_largest_head_count_fits_the_kernels_offsets():
    """2^19 heads of 256 bytes, and the last of a block's 16 rows at the largest stride (2^26 - 8 elements)."""
    heads, stride = 2**19, 2**26 - 8
    assert 2 * 128 * heads < 2**31 and 2 * (15 * stride + heads * 128) <= 2**31 - 1


@pytest.mark.parametrize("pages,hkv,page", [(3, 1, 16), (1, 1, 8), (5, 3, 24), (4, 2, 16), (0, 1, 16)])
def test_scale_bytes_come_in_whole_words(pages, hkv, page):
    """The decode reads the word around a block's pair of bytes: behind an odd number of pairs that is memory, too."""
    import pa_amd
    s = pa_amd.alloc_kv_scales(pages, hkv, page, device="cpu")
    assert s.shape == (pages, hkv, page // pa_amd.block_tokens(page), 2) and s.is_contiguous() and bool((s == 127).all())
    assert s.untyped_storage().nbytes() % 4 == 0 and s.storage_offset() == 0


class _OnDevice:
    """What the checks ask of a CUDA tensor."""

    def __init__(self, shape, device):
        self.shape, self.device_index, self.is_cuda = shape, device, True

    def get_device(self):
        return self.device_index

    def is_contiguous(self):
        return True

    def element_size(self):
        return 1

    def size(self, i):
        return self.shape[i]


def test_scales_of_another_device_are_refused():
    """The decode's caches and scales lie on one device. (The compiled binding makes the same check; two devices are not
    at hand.)"""
    from pa_amd import ops
    cache = _OnDevice((6, 2, 16, 128), 1)
    ops.check_kv_scales(_OnDevice((6, 2, 1, 2), 1), cache)
    with pytest.raises(RuntimeError, match="device"):
        ops.check_kv_scales(_OnDevice((6, 2, 1, 2), 0), cache)
