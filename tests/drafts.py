"""Plain implementations, in 64 bits on the CPU, of attention of drafted tokens over a paged cache, of keeping accepted
rows and of reading rows back, and the caches that their tests use. Written from the operators' definitions
(include/pa_decode.h)."""

from __future__ import annotations

import math

import numpy as np
import torch

from new_tokens import e4m3, e4m3_encode

D = 128


def block_of(page: int) -> int:
    return 16 if page % 16 == 0 else 8


class Cache:
    """A paged cache with random rows in every place and pages in random order: raw arrays on the CPU (numpy) and the
    device's copies. kind: fp16, fp8 or block. rows x cols: the block table, every entry a page of its own."""

    def __init__(self, kind, page, hkv, rows, cols, seed=0, k_scale=0.02, v_scale=0.03, spare=2):
        r = np.random.default_rng(seed)
        self.kind, self.page, self.hkv = kind, page, hkv
        self.pages = rows * cols + spare
        shape = (self.pages, hkv, page, D)
        self.k_scale = self.v_scale = 1.0
        self.scales = None
        if kind == "fp16":
            self.kv = [r.standard_normal(shape).astype(np.float16) for _ in range(2)]
        else:
            self.kv = [e4m3_encode(r.standard_normal(shape) * 40.0) for _ in range(2)]
            if kind == "fp8":
                self.k_scale, self.v_scale = float(np.float32(k_scale)), float(np.float32(v_scale))
            else:
                self.scales = r.integers(119, 125, (self.pages, hkv, page // block_of(page), 2)).astype(np.uint8)
        self.table = r.permutation(self.pages)[:rows * cols].reshape(rows, cols).astype(np.int32)

    def device(self):
        """The arrays as tensors on the device: k, v, table, scales (None without)."""
        k, v = (torch.from_numpy(x.copy()).cuda() for x in self.kv)
        return k, v, torch.from_numpy(self.table.copy()).cuda(), (
            None if self.scales is None else torch.from_numpy(self.scales.copy()).cuda())

    def kw(self, scales):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale, "kv_scales": scales}

    def values(self, j, page, slot):
        """Row [hkv, 128] of the keys (j = 0) or values as numbers."""
        x = self.kv[j][page, :, slot]
        if self.kind == "fp16":
            return x.astype(np.float64)
        x = e4m3(x)
        if self.kind == "fp8":
            return x * (self.v_scale if j else self.k_scale)
        e = self.scales[page, :, slot // block_of(self.page), j].astype(np.float64)
        return x * np.exp2(e - 127.0)[:, None]

    def rows(self, j, row, lo, hi):
        """Places lo .. hi - 1 of a table row, [places, hkv, 128]; pages out of range hold zeros."""
        out = np.zeros((hi - lo, self.hkv, D))
        for i, pos in enumerate(range(lo, hi)):
            page = int(self.table[row, pos // self.page])
            if 0 <= page < self.pages:
                out[i] = self.values(j, page, pos % self.page)
        return out


def tree_bits(tree, words):
    """Rows of a tree given as whole numbers (bit j: token j), int64 [tokens, words]."""
    flat = [[(x >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for x in tree]
    return torch.from_numpy(np.array(flat, dtype=np.uint64).reshape(len(tree), words).view(np.int64).copy()).cuda()


def random_tree(r, n, spread=6):
    rows = []
    for i in range(n):
        up = int(r.integers(max(-1, i - spread), i)) if i else -1
        rows.append((1 << i) | (rows[up] if up >= 0 else 0))
    return rows


# A score's error before the exponential, relative to sm_scale sum |q k|: 128 products of fp16 values, exact in 32 bits,
# summed in 32 bits in any order, 2^-17 at most; its scaling and the exponent's argument 2^-22 more.
SCORE_REL = 2.0 ** -17 + 2.0 ** -22


def attention(q, k, v, seen, scale):
    """q [n, hq, 128], k and v [places, hkv, 128], seen [n, places] -> (result [n, hq, 128], its tolerance).
    Tolerance: a probability is off by 2^-11 (fp16) and its score's error, twice (it is in the denominator, too), and
    by 2^-31 of the largest where it is subnormal in fp16; sums in 32 bits of `places` terms, in runs of 16 (and as
    many joins as that at most); the values' own rounding where a block's scale makes them fp16 subnormals, 2^-25;
    the result's rounding."""
    n, hq, _ = q.shape
    hkv = k.shape[1]
    out, tol = np.zeros((n, hq, D)), np.full((n, hq, D), 2.0 ** -24)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = scale * (q[:, h] @ kh.T)
        err = SCORE_REL * abs(scale) * (np.abs(q[:, h]) @ np.abs(kh).T)
        for i in range(n):
            m = seen[i]
            if not m.any():
                continue
            p = np.exp(s[i, m] - s[i, m].max())
            p /= p.sum()
            out[i, h] = p @ vh[m]
            size = p @ np.abs(vh[m])
            rel = 2.0 ** -11 + 2.0 * err[i, m].max() + (m.sum() / 8 + 64) * 2.0 ** -24
            tol[i, h] += size * rel * 1.01 + np.abs(out[i, h]) * 2.0 ** -11 + np.abs(vh[m]).sum(0) * 2.0 ** -31 * p.max()
    return out, tol


def seen_of(start, n, tree):
    """Which places 0 .. start + n - 1 an entry's tokens see; tree None: a chain."""
    new = np.tril(np.ones((n, n), bool)) if tree is None else np.array(
        [[(row >> j) & 1 for j in range(n)] for row in tree], dtype=bool).reshape(n, n)
    return np.concatenate([np.ones((n, start), bool), new], axis=1)


def need(amax):
    """Smallest k in [-32, 8] with amax <= 448 * 2^k."""
    k = -32
    while k < 8 and amax > 448.0 * 2.0 ** k:
        k += 1
    return k


def keep(cache: Cache, entries):
    """entries: (row, start, kept numbers in order). Moves rows of cache.kv and cache.scales in place."""
    P = cache.page

    def spot(row, pos):
        i = pos // P
        if not 0 <= row < cache.table.shape[0] or i >= cache.table.shape[1] or pos < 0:
            return None
        page = int(cache.table[row, i])
        return (page, pos % P) if 0 <= page < cache.pages else None
    for row, start, kept in entries:
        moves = [(j, k, spot(row, start + k), spot(row, start + j)) for j, k in enumerate(kept)]
        moves = [m for m in moves if m[1] >= m[0] and m[2] is not None and m[3] is not None]
        for v in range(2):
            pool = cache.kv[v]
            if cache.kind != "block":
                took = [pool[s[0], :, s[1]].copy() for _, _, s, _ in moves]
                for x, (_, _, _, d) in zip(took, moves):
                    pool[d[0], :, d[1]] = x
                continue
            B = block_of(P)
            was = {s: (pool[s[0], :, s[1]].copy(), cache.values(v, *s)) for _, _, s, _ in moves}
            for b in sorted({(start + j) // B for j, _, _, _ in moves}):
                mine = [m for m in moves if (start + m[0]) // B == b]
                if all(j == k for j, k, _, _ in mine):
                    continue
                page, s0 = spot(row, b * B)
                for h in range(cache.hkv):
                    old = int(cache.scales[page, h, s0 // B, v]) - 127
                    vals = np.stack([was[m[2]][1][h] for m in mine])
                    big = np.nanmax(np.abs(vals)) if not np.isnan(vals).all() else 0.0
                    k = need(big)
                    top = lambda k: 240.0 if k == 8 else 448.0
                    if b * B < start:
                        k = max(k, old)
                        if k > old:
                            for s in range(s0, s0 + start - b * B):
                                code = pool[page, h, s]
                                new = e4m3_encode(e4m3(code) * 2.0 ** (old - k), top(k))
                                pool[page, h, s] = np.where((code & 0x7f) == 0x7f, code, new)
                    for _, _, s, d in mine:
                        code, x = was[s][0][h], was[s][1][h]
                        pool[d[0], h, d[1]] = np.where((code & 0x7f) == 0x7f, code, e4m3_encode(x * 2.0 ** -k, top(k)))
                    cache.scales[page, h, s0 // B, v] = k + 127
