"""New tokens of a step on torch tensors: head norms with rotation, appends with
rotation into caller-owned paged caches (pa_norm_rope, pa_append_rope), and what
drafted tokens need there: attention of several tokens per sequence (pa_tree_attention),
accepted rows kept (pa_keep_rows), rows read back (pa_read_cache).

    rope = Rope(freqs)                                   # a model's rotation, made once
    q, k = norm_rope(q, k, positions, rope, q_weight=wq, k_weight=wk)
    q = append_rope(q, k, v, k_cache, v_cache, block_table, tok_begin, start_pos, rope, ...)
    out = tree_attention(q, k_cache, v_cache, block_table, tok_begin, start_pos, tree, ...)
    keep_rows(k_cache, v_cache, block_table, kept, counts, start_pos, ...)
    k, v = read_cache(k_cache, v_cache, block_table, tok_begin, start_pos, num_tokens, ...)

They run on the current torch stream of the tensors' device, through the compiled
binding where it was built, else through ctypes. Argument errors raise
RuntimeError (as Decoder's do) or the library's errors; nothing is differentiated.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib
from ._lib import AppendArgs, CachedTokens, HeadRows, InvalidArgument, call, check, load
from .decoder import _current_stream, _require, compiled

D = 128


def block_tokens(page_size: int) -> int:
    """Tokens per block of a block-scaled cache: 16 or 8, 0 for page sizes it does not take."""
    return load().pa_block_tokens(page_size)


def alloc_kv_scales(num_pages: int, num_kv_heads: int, page_size: int, device=None) -> torch.Tensor:
    """Scale bytes of a block-scaled cache ([pages][kv heads][blocks of a page][2]; byte e
    stands for 2^(e - 127)). What is in them before a block's first token does not matter.
    The memory is rounded up to whole 4-byte words, which the decode reads."""
    b = block_tokens(page_size)
    if b == 0:
        raise InvalidArgument("block-scaled caches need a page_size that is a multiple of 8")
    shape = (num_pages, num_kv_heads, page_size // b, 2)
    n = math.prod(shape)
    flat = torch.full(((n + 3) // 4 * 4,), 127, dtype=torch.uint8, device=device if device is not None else "cuda")
    return flat[:n].view(shape)


class Rope:
    """A model's rotation on one device (pa_rope): pair i turns by freqs[i] radians per
    position. freqs: rot_dim / 2 numbers (rot_dim, a multiple of 16 up to 128, leading
    dims turn). Pairs are dims (i, i + rot_dim / 2), or (2i, 2i + 1) if interleaved.
    axes: which of a token's positions turns pair i, for tokens with several. scale
    multiplies the sines and cosines. Kept as long as calls and graphs that use it run."""

    def __init__(self, freqs, axes=None, interleaved: bool = False, scale: float = 1.0, num_axes: int | None = None,
                 device=None):
        f = freqs.detach().cpu().numpy() if hasattr(freqs, "detach") else freqs
        f = np.ascontiguousarray(f, dtype=np.float64)
        a = None
        if axes is not None:
            a = axes.detach().cpu().numpy() if hasattr(axes, "detach") else axes
            a = np.ascontiguousarray(a, dtype=np.int32)
        if f.ndim != 1 or (a is not None and a.shape != f.shape):
            raise InvalidArgument("rope: freqs and axes must be 1-D of one length")
        self.rot_dim = 2 * f.size
        if num_axes is None:
            num_axes = 1 if a is None or a.size == 0 else int(a.max()) + 1
        self.num_axes = int(num_axes)
        self.handle = 0
        h = ctypes.c_void_p()
        load()
        index = None if device is None else torch.device(device).index
        with torch.cuda.device(index):   # None: no change
            call("pa_rope_create", f.ctypes.data, None if a is None else a.ctypes.data, self.rot_dim, self.num_axes,
                 int(interleaved), float(scale), ctypes.byref(h))
        self.handle = h.value

    def __del__(self):
        try:
            if self.handle:
                load().pa_rope_destroy(self.handle)
                self.handle = 0
        except Exception:
            pass


def _heads_ok(x, n: int) -> bool:
    return (x.is_cuda and x.dtype == torch.float16 and x.dim() == 3 and x.size(0) == n and x.size(1) > 0
            and x.size(2) == D and x.stride(2) == 1 and (x.size(1) == 1 or x.stride(1) == D))


def _row_stride(x) -> int:
    return x.stride(0) if x.size(0) > 1 else x.size(1) * D


def head_rows(name: str, x, weight, eps: float, out=None, device=None) -> HeadRows:
    """pa_head_rows of a [tokens, heads, 128] tensor, checked as the compiled binding does."""
    _require(_heads_ok(x, x.size(0) if x.dim() else 0) and (device is None or x.get_device() == device),
             f"{name} must be a CUDA fp16 [tokens, heads, 128] tensor whose heads are contiguous")
    r = HeadRows()
    r.in_, r.in_stride, r.heads, r.eps = x.data_ptr(), _row_stride(x), x.size(1), float(eps)
    if weight is not None:
        _require(weight.is_cuda and weight.get_device() == x.get_device() and weight.dtype == torch.float32
                 and weight.is_contiguous() and weight.numel() == D,
                 f"{name}_weight must be a contiguous CUDA float32 tensor of 128")
        r.weight = weight.data_ptr()
    if out is not None:
        _require(_heads_ok(out, x.size(0)) and out.get_device() == x.get_device() and out.size(1) == x.size(1),
                 f"{name}_out must be a CUDA fp16 tensor of the shape of {name} whose heads are contiguous")
        r.out, r.out_stride = out.data_ptr(), _row_stride(out)
    return r


def positions_ptr(positions, rope, n: int, device: int):
    if positions is None:
        return None
    axes = rope.num_axes if rope is not None else positions.numel() // max(n, 1)
    _require(positions.is_cuda and positions.get_device() == device and positions.dtype == torch.int32
             and positions.is_contiguous() and positions.numel() == n * axes
             and (positions.dim() == 1 or (positions.dim() == 2 and positions.size(0) == n)),
             "positions must be a contiguous CUDA int32 [tokens] or [tokens, axes] tensor")
    return positions.data_ptr()


def norm_rope(q, k, positions, rope: Rope | None = None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
              q_out=None, k_out=None):
    """Heads of q [n, Hq, 128] and k [n, Hkv, 128] (fp16; one may be None) RMS-normed over
    their 128 dims (where a float32 weight is given) and rotated to positions (int32 [n], or
    [n, axes]; None only without rope), in one pass. Tokens may be strided (a fused projection's
    columns), heads are contiguous. Returns (q_out, k_out); an output may be its input."""
    c = compiled()
    if c is not None:
        return c.norm_rope(q, k, positions, 0 if rope is None else rope.handle, q_weight, k_weight, eps, q_out, k_out)
    _require(q is not None or k is not None, "q or k is needed")
    x = q if q is not None else k
    _require(x.is_cuda and x.dim() == 3, "q and k must be CUDA fp16 [tokens, heads, 128] tensors")
    n, dev = x.size(0), x.get_device()
    _require(n < 2**31, "too many tokens")
    rows = []
    for name, t, w, out in (("q", q, q_weight, q_out), ("k", k, k_weight, k_out)):
        if t is None:
            rows.append((None, None))
            continue
        _require(t.dim() == 3 and t.size(0) == n, f"{name} must be a CUDA fp16 [tokens, heads, 128] tensor whose heads are contiguous")
        out = torch.empty((n, t.size(1), D), dtype=torch.float16, device=t.device) if out is None else out
        rows.append((head_rows(name, t, w, eps, out, dev), out))
    pos = positions_ptr(positions, rope, n, dev)
    with torch.cuda.device(dev):
        check(load().pa_norm_rope(None if rope is None else rope.handle,
                                  *(None if r is None else ctypes.byref(r) for r, _ in rows), pos, n,
                                  _current_stream(dev)))
    return rows[0][1], rows[1][1]


def append_rope(q, k, v, k_cache, v_cache, block_table, tok_begin, start_pos, rope: Rope | None = None, *,
                positions=None, q_weight=None, k_weight=None, eps: float = 1e-6, k_scale: float = 1.0,
                v_scale: float = 1.0, kv_scales=None, slot_ids=None, q_out=None):
    """New tokens of several sequences into a caller's paged cache, in one launch: k [n, Hkv, 128]
    normed (k_weight) and rotated (rope) into the pages, v as it is, q (or None) normed and
    rotated into q_out. Entry e holds tokens tok_begin[e] .. tok_begin[e + 1] - 1 (device int32
    [entries + 1]); they go to places start_pos[e], start_pos[e] + 1, ... (device int32 [entries])
    of the sequence whose pages block_table[slot_ids[e]] lists (row e without slot_ids). positions:
    what the rotation takes in place of the tokens' places ([n] or [n, axes]). Caches: fp16, or
    one-byte FP8 with k_scale / v_scale (a code c stands for c * scale), or with kv_scales (alloc_kv_scales)
    block-scaled, where one call holds each sequence once. Tokens whose place, row or page is
    out of range, or that are in no entry (padding), are left out. Returns q_out (None without q)."""
    c = compiled()
    if c is not None:
        return c.append_rope(q, k, v, k_cache, v_cache, block_table, tok_begin, start_pos,
                             0 if rope is None else rope.handle, positions, q_weight, k_weight, eps, k_scale, v_scale,
                             kv_scales, slot_ids, q_out)
    _require(k.is_cuda and k.dim() == 3, "k must be a CUDA fp16 [tokens, heads, 128] tensor")
    n, dev, hkv = k.size(0), k.get_device(), k.size(1)
    _require(n < 2**31, "too many tokens")
    qr = None
    if q is not None:
        _require(q.dim() == 3 and q.size(0) == n, "q must be a CUDA fp16 [tokens, heads, 128] tensor whose heads are contiguous")
        q_out = torch.empty((n, q.size(1), D), dtype=torch.float16, device=q.device) if q_out is None else q_out
        qr = head_rows("q", q, q_weight, eps, q_out, dev)
    kr = head_rows("k", k, k_weight, eps, None, dev)
    _require(_heads_ok(v, n) and v.get_device() == dev and v.size(1) == hkv,
             "v must be a CUDA fp16 tensor of k's shape whose heads are contiguous")
    for x in (k_cache, v_cache):
        _require(x.is_cuda and x.get_device() == dev and x.is_contiguous() and x.dim() == 4 and x.size(1) == hkv
                 and x.size(2) > 0 and x.size(3) == D and x.shape == k_cache.shape and x.dtype == k_cache.dtype
                 and (x.dtype == torch.float16 or x.element_size() == 1),
                 "k_cache and v_cache must be contiguous CUDA [pages, k's heads, page_size, 128] tensors, both fp16 "
                 "or both one-byte FP8")
    fp16 = k_cache.dtype == torch.float16
    _require(kv_scales is None or not fp16, "kv_scales goes with one-byte FP8 caches")
    if kv_scales is not None:
        check_kv_scales(kv_scales, k_cache)

    def ints(t, size, what):
        _require(t.is_cuda and t.get_device() == dev and t.dtype == torch.int32 and t.is_contiguous() and t.dim() == 1
                 and (size is None or t.size(0) == size), what)
        return t.data_ptr()
    a = AppendArgs()
    a.num_tokens = n
    a.start_pos = ints(start_pos, None, "start_pos must be a contiguous CUDA int32 [entries] tensor")
    m = a.num_entries = start_pos.size(0)
    a.tok_begin = ints(tok_begin, m + 1, "tok_begin must be a contiguous CUDA int32 [entries + 1] tensor")
    if slot_ids is not None:
        a.slot_ids = ints(slot_ids, m, "slot_ids must be a contiguous CUDA int32 [entries] tensor")
    _require(block_table.is_cuda and block_table.get_device() == dev and block_table.dtype == torch.int32
             and block_table.is_contiguous() and block_table.dim() == 2 and block_table.size(1) > 0,
             "block_table must be a contiguous CUDA int32 [rows, columns] tensor")
    a.positions = positions_ptr(positions, rope, n, dev)
    a.v, a.v_stride = v.data_ptr(), _row_stride(v)
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.kv_scales = None if kv_scales is None else kv_scales.data_ptr()
    a.block_table, a.block_table_stride, a.num_table_rows = block_table.data_ptr(), block_table.size(1), block_table.size(0)
    a.num_pages, a.page_size, a.k_scale, a.v_scale = k_cache.size(0), k_cache.size(2), float(k_scale), float(v_scale)
    dtype = _lib.PA_KV_FP16 if fp16 else _lib.PA_KV_FP8_E4M3 if kv_scales is None else _lib.PA_KV_FP8_E4M3_BLOCK
    with torch.cuda.device(dev):
        check(load().pa_append_rope(dtype, ctypes.byref(a), None if rope is None else rope.handle,
                                    None if qr is None else ctypes.byref(qr), ctypes.byref(kr), _current_stream(dev)))
    return q_out


def _cached_tokens(k_cache, v_cache, block_table, tok_begin, start_pos, k_scale, v_scale, kv_scales, slot_ids, n: int):
    """pa_cached_tokens of n tokens (tok_begin None: none), checked as the compiled binding does, and the cache's type."""
    dev = k_cache.get_device() if k_cache.is_cuda else -1
    for x in (k_cache, v_cache):
        _require(x.is_cuda and x.get_device() == dev and x.is_contiguous() and x.dim() == 4 and x.size(1) > 0
                 and x.size(2) > 0 and x.size(3) == D and x.shape == k_cache.shape and x.dtype == k_cache.dtype
                 and (x.dtype == torch.float16 or x.element_size() == 1),
                 "k_cache and v_cache must be contiguous CUDA [pages, kv heads, page_size, 128] tensors, both fp16 "
                 "or both one-byte FP8")
    fp16 = k_cache.dtype == torch.float16
    _require(kv_scales is None or not fp16, "kv_scales goes with one-byte FP8 caches")
    if kv_scales is not None:
        check_kv_scales(kv_scales, k_cache)

    def ints(t, size, what):
        _require(t.is_cuda and t.get_device() == dev and t.dtype == torch.int32 and t.is_contiguous() and t.dim() == 1
                 and (size is None or t.size(0) == size), what)
        return t.data_ptr()
    _require(0 <= n < 2**31, "too many tokens")
    c = CachedTokens()
    c.num_tokens = n
    c.start_pos = ints(start_pos, None, "start_pos must be a contiguous CUDA int32 [entries] tensor")
    m = c.num_entries = start_pos.size(0)
    if tok_begin is not None:
        c.tok_begin = ints(tok_begin, m + 1, "tok_begin must be a contiguous CUDA int32 [entries + 1] tensor")
    if slot_ids is not None:
        c.slot_ids = ints(slot_ids, m, "slot_ids must be a contiguous CUDA int32 [entries] tensor")
    _require(block_table.is_cuda and block_table.get_device() == dev and block_table.dtype == torch.int32
             and block_table.is_contiguous() and block_table.dim() == 2 and block_table.size(1) > 0,
             "block_table must be a contiguous CUDA int32 [rows, columns] tensor")
    c.k_cache, c.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    c.kv_scales = None if kv_scales is None else kv_scales.data_ptr()
    c.block_table, c.block_table_stride, c.num_table_rows = block_table.data_ptr(), block_table.size(1), block_table.size(0)
    c.num_pages, c.num_kv_heads, c.page_size = k_cache.size(0), k_cache.size(1), k_cache.size(2)
    c.k_scale, c.v_scale = float(k_scale), float(v_scale)
    return c, _lib.PA_KV_FP16 if fp16 else _lib.PA_KV_FP8_E4M3 if kv_scales is None else _lib.PA_KV_FP8_E4M3_BLOCK


def tree_rows(parents, device=None) -> torch.Tensor:
    """tree_attention's `tree` for drafted trees given by their tokens' parents: parents[e][i] is the number within
    entry e of the token that its token i continues, below i, or -1 where it continues the sequence itself. Returns
    int64 [tokens of all entries, words of the largest], a token's bits being its own and its ancestors'."""
    words = max([1] + [(len(p) + 63) // 64 for p in parents])
    out = np.zeros((sum(len(p) for p in parents), words), dtype=np.uint64)
    at = 0
    for p in parents:
        for i, up in enumerate(p):
            up = int(up)
            if not -1 <= up < i:
                raise InvalidArgument("tree_rows: a token's parent comes before it (-1: the sequence itself)")
            if up >= 0:
                out[at + i] = out[at + up]
            out[at + i, i // 64] |= np.uint64(1 << (i % 64))
        at += len(p)
    return torch.from_numpy(out.view(np.int64)).to(device if device is not None else "cuda")


def tree_attention(q, k_cache, v_cache, block_table, tok_begin, start_pos, tree=None, *, k_scale: float = 1.0,
                   v_scale: float = 1.0, kv_scales=None, slot_ids=None, sm_scale: float | None = None, out=None):
    """Attention of several new tokens per sequence, all of them in the paged cache already, over their sequences:
    q [n, Hq, 128] fp16 -> out [n, Hq, 128] (Hq up to 32 times the cache's heads; tokens may be strided). Entry e holds tokens
    tok_begin[e] .. tok_begin[e + 1] - 1 (device int32 [entries + 1]), whose keys and values lie at places start_pos[e],
    start_pos[e] + 1, ... of the sequence whose pages block_table[slot_ids[e]] lists (row e without slot_ids). Token i
    of an entry sees every place before start_pos[e] and, of the entry's tokens, those whose bits its row of tree
    (int64 [n, words]; tree_rows makes it) has, or without tree itself and those before it: a chain, a piece of a
    prompt. Caches as append_rope's. sm_scale: 1 / sqrt(128) unless given. A token that sees nothing gets zeros;
    tokens of no entry (padding), or of one out of range, keep what out held; out may be q. Returns out."""
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    c = compiled()
    if c is not None:
        return c.tree_attention(q, k_cache, v_cache, block_table, tok_begin, start_pos, tree, k_scale, v_scale,
                                kv_scales, slot_ids, scale, out)
    _require(q.is_cuda and q.dim() == 3, "q must be a CUDA fp16 [tokens, heads, 128] tensor")
    n, dev = q.size(0), q.get_device()
    a, dtype = _cached_tokens(k_cache, v_cache, block_table, tok_begin, start_pos, k_scale, v_scale, kv_scales, slot_ids, n)
    _require(k_cache.get_device() == dev, "q and the caches must be on one device")
    out = torch.empty((n, q.size(1), D), dtype=torch.float16, device=q.device) if out is None else out
    r = head_rows("q", q, None, 0.0, out, dev)
    if tree is not None:
        _require(tree.is_cuda and tree.get_device() == dev and tree.dtype == torch.int64 and tree.is_contiguous()
                 and tree.dim() == 2 and tree.size(0) == n and tree.size(1) > 0,
                 "tree must be a contiguous CUDA int64 [tokens, words] tensor")
    with torch.cuda.device(dev):
        need = ctypes.c_size_t()
        check(load().pa_tree_attention_workspace(dtype, ctypes.byref(a), q.size(1), ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        check(load().pa_tree_attention(dtype, ctypes.byref(a), ctypes.byref(r), None if tree is None else tree.data_ptr(),
                                       0 if tree is None else tree.size(1), scale, None if ws is None else ws.data_ptr(),
                                       need.value, _current_stream(dev)))
    return out


_VALUE_TYPES = {torch.float16: _lib.PA_VALUE_FP16, torch.bfloat16: _lib.PA_VALUE_BF16, torch.float32: _lib.PA_VALUE_FP32}


def read_cache(k_cache, v_cache, block_table, tok_begin, start_pos, num_tokens: int, *, dtype=torch.float16,
               k_scale: float = 1.0, v_scale: float = 1.0, kv_scales=None, slot_ids=None, k_out=None, v_out=None):
    """Rows of a paged cache as numbers: token t of num_tokens (those of the last entry and any padding behind) of
    entry e, the place start_pos[e] + t - tok_begin[e] of its sequence, to k_out[t] and v_out[t] ([n, Hkv, 128] of
    dtype: float16, bfloat16 or float32; tokens may be strided). Entries, tables and caches as tree_attention's. Tokens
    of no entry, and those whose place, row or page is out of range, keep what the outputs held. Returns (k_out, v_out)."""
    _require(dtype in _VALUE_TYPES, "dtype must be float16, bfloat16 or float32")
    c = compiled()
    if c is not None:
        return c.read_cache(k_cache, v_cache, block_table, tok_begin, start_pos, num_tokens, _VALUE_TYPES[dtype], k_scale,
                            v_scale, kv_scales, slot_ids, k_out, v_out)
    a, cache = _cached_tokens(k_cache, v_cache, block_table, tok_begin, start_pos, k_scale, v_scale, kv_scales, slot_ids,
                              num_tokens)
    dev = k_cache.get_device()
    outs = []
    for x in (k_out, v_out):
        x = torch.empty((num_tokens, k_cache.size(1), D), dtype=dtype, device=k_cache.device) if x is None else x
        _require(x.is_cuda and x.get_device() == dev and x.dtype == dtype and x.dim() == 3 and x.size(0) == num_tokens
                 and x.size(1) == k_cache.size(1) and x.size(2) == D and x.stride(2) == 1
                 and (x.size(1) == 1 or x.stride(1) == D),
                 "k_out and v_out must be CUDA [tokens, kv heads, 128] tensors of the dtype asked for, their heads contiguous")
        outs.append(x)
    with torch.cuda.device(dev):
        check(load().pa_read_cache(cache, ctypes.byref(a), _VALUE_TYPES[dtype], outs[0].data_ptr(), _row_stride(outs[0]),
                                   outs[1].data_ptr(), _row_stride(outs[1]), _current_stream(dev)))
    return outs[0], outs[1]


def keep_rows(k_cache, v_cache, block_table, kept, counts, start_pos, *, kv_scales=None, slot_ids=None) -> None:
    """Accepted drafted tokens up in their sequences, in place: of the rows at places start_pos[e], start_pos[e] + 1,
    ... those with the numbers kept[e][0] < ... < kept[e][counts[e] - 1] (device int32 [entries, width] and [entries])
    go to places start_pos[e], start_pos[e] + 1, ... of their sequence. Each sequence once a call. Rows past the last
    kept one keep their bytes. In block-scaled caches the blocks that a row moves into get the scale that their kept
    rows ask for, as an append chooses it."""
    c = compiled()
    if c is not None:
        return c.keep_rows(k_cache, v_cache, block_table, kept, counts, start_pos, kv_scales, slot_ids)
    a, cache = _cached_tokens(k_cache, v_cache, block_table, None, start_pos, 1.0, 1.0, kv_scales, slot_ids, 0)
    dev = k_cache.get_device()
    _require(kept.is_cuda and kept.get_device() == dev and kept.dtype == torch.int32 and kept.is_contiguous()
             and kept.dim() == 2 and kept.size(0) == a.num_entries, "kept must be a contiguous CUDA int32 [entries, width] tensor")
    _require(counts.is_cuda and counts.get_device() == dev and counts.dtype == torch.int32 and counts.is_contiguous()
             and counts.dim() == 1 and counts.size(0) == a.num_entries, "counts must be a contiguous CUDA int32 [entries] tensor")
    with torch.cuda.device(dev):
        check(load().pa_keep_rows(cache, ctypes.byref(a), kept.data_ptr(), kept.size(1), counts.data_ptr(),
                                  _current_stream(dev)))


def check_kv_scales(s, cache) -> None:
    b = block_tokens(cache.size(2))
    _require(b != 0, "block-scaled caches need a page_size that is a multiple of 8")
    _require(s.is_cuda and s.get_device() == cache.get_device() and s.is_contiguous() and s.element_size() == 1
             and tuple(s.shape) == (cache.size(0), cache.size(1), cache.size(2) // b, 2),
             f"kv_scales must be a contiguous CUDA uint8 [pages, num_kv_heads, page_size / {b}, 2] tensor on the "
             "cache's device")
