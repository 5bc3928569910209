"""Plain implementations of the new-token operators in 64 bits, for the tests: head norms with rotation, and what a
block-scaled cache holds after a history of appends. Written from the operators' definitions (include/pa_decode.h)."""

from __future__ import annotations

import numpy as np

import oracle

D = 128


def freqs(rot: int, theta: float = 10000.0) -> np.ndarray:
    return theta ** (-2.0 * np.arange(rot // 2) / rot)


def norm_rotate(x, weight, eps, pos, fr, axes=None, interleaved=False, scale=1.0):
    """x [n, h, 128] float64, pos [n, axes] int64 -> (result, what it is computed from: |a| + |b| of each dim's pair).
    Angles in 80 bits: a place of 2^31 turns by that many radians."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x * np.asarray(weight, np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    mag = np.abs(x)
    if fr is None:
        return x, mag
    m = len(fr)
    pos = np.asarray(pos, np.int64).reshape(x.shape[0], -1)
    at = pos[:, np.zeros(m, int) if axes is None else np.asarray(axes)].astype(np.longdouble)
    angle = at * np.asarray(fr, np.longdouble)
    c = (scale * np.cos(angle)).astype(np.float64)[:, None]
    s = (scale * np.sin(angle)).astype(np.float64)[:, None]
    y = x.copy()
    lo, hi = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if interleaved else (slice(0, m), slice(m, 2 * m))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    mag[..., lo] = mag[..., hi] = abs(scale) * (np.abs(a) + np.abs(b))
    return y, mag


# A result in 32 bits before its one rounding, relative to |a| + |b|: the norm's sum of 128 squares (4 + 7 additions
# deep, halved by the root), root, quotient and two products, 2^-20.7; sine and cosine and their argument (of 2^31 turns
# at most), 2^-20.4; two products and their sum, 2^-23. Together below 2^-19.
F32_REL = 2.0 ** -19


def f16_tol(ref, mag):
    """Half an fp16 step of the result (2^-11 of it, 2^-25 where it is subnormal) on top of the 32-bit error."""
    return np.abs(ref) * 2.0 ** -11 * (1 + 2.0 ** -10) + mag * F32_REL + 2.0 ** -25


def e4m3_tol(ref, mag, scale):
    """Half an E4M3 step: 2^-4 of the value, 2^-10 of the scale where it is subnormal."""
    return np.maximum((np.abs(ref) + mag * F32_REL) * 2.0 ** -4, scale * 2.0 ** -10) + mag * F32_REL


def f16(bits: np.ndarray) -> np.ndarray:
    return np.asarray(bits, np.uint16).view(np.float16).astype(np.float64)


_DECODED = None


def e4m3(codes: np.ndarray) -> np.ndarray:
    global _DECODED
    if _DECODED is None:
        _DECODED = oracle.e4m3_to_f32(np.arange(256)).astype(np.float64)
    return _DECODED[np.asarray(codes, np.uint8)]


def e4m3_encode(x: np.ndarray, top: float = 448.0) -> np.ndarray:
    """Round to nearest even, saturating at top; a NaN keeps its sign. From the table of all codes: the nearest one,
    the even one of two."""
    x = np.asarray(x, np.float64)
    table = e4m3(np.arange(127))                      # 0 .. 448, rising with the code
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), top)
    i = np.searchsorted(table, a).clip(1, 126)
    lo, hi = a - table[i - 1], table[i] - a
    code = np.where(lo < hi, i - 1, np.where(hi < lo, i, np.where(i % 2 == 0, i, i - 1)))
    code = np.where(np.isnan(x), 0x7F, code)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def block_tokens(page: int) -> int:
    return 16 if page % 16 == 0 else 8


def exponent(amax: float) -> int:
    """The smallest k in [-32, 8] with amax <= 448 * 2^k."""
    for k in range(-32, 8):
        if amax <= 448.0 * 2.0 ** k:
            return k
    return 8


class BlockPool:
    """What one pool (K or V) of a block-scaled cache holds: codes [pages, hkv, P, 128], scale exponents."""

    def __init__(self, codes: np.ndarray, scale_bytes: np.ndarray):
        self.codes, self.exps = codes.copy(), scale_bytes.astype(np.int64) - 127
        self.P = codes.shape[2]
        self.B = block_tokens(self.P)

    def append(self, x: np.ndarray, start: int, table) -> None:
        """x [n, hkv, 128] float64 to places start .. start + n - 1 of the sequence with these pages, in one call."""
        n, hkv, B, P = x.shape[0], x.shape[1], self.B, self.P
        for blk in range(start // B, (start + n - 1) // B + 1 if n else start // B):
            lo, hi = max(start, blk * B), min(start + n, (blk + 1) * B)
            page, b, s0 = table[blk * B // P], blk * B % P // B, blk * B % P
            rows = slice(s0 + lo % B, s0 + lo % B + hi - lo)
            for h in range(hkv):
                part = x[lo - start:hi - start, h]
                a = np.abs(part[~np.isnan(part)])
                k = exponent(a.max() if a.size else 0.0)
                if lo % B:
                    was = self.exps[page, h, b]
                    if k > was:
                        old = self.codes[page, h, s0:s0 + lo % B]
                        new = e4m3_encode(e4m3(old) * 2.0 ** float(was - k), 240.0 if k == 8 else 448.0)
                        self.codes[page, h, s0:s0 + lo % B] = np.where((old & 0x7F) == 0x7F, old, new)
                    k = max(k, was)
                self.exps[page, h, b] = k
                self.codes[page, h, rows] = e4m3_encode(part * 2.0 ** -float(k), 240.0 if k == 8 else 448.0)

    def values(self) -> np.ndarray:
        """[pages, hkv, P, 128] float64."""
        return e4m3(self.codes) * np.repeat(2.0 ** self.exps, self.B, axis=2)[..., None]


def attention(q, k, v):
    """q [Hq, 128], k and v [L, Hkv, 128] float64 -> (out, sum of p |v|, largest sum of |q k|)."""
    hkv = k.shape[1]
    G = q.shape[0] // hkv
    out, weight, big = np.empty_like(q), np.empty_like(q), 0.0
    for h in range(hkv):
        qh = q[h * G:(h + 1) * G]
        s = qh @ k[:, h].T / np.sqrt(128.0)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[h * G:(h + 1) * G] = p @ v[:, h]
        weight[h * G:(h + 1) * G] = p @ np.abs(v[:, h])
        big = max(big, float((np.abs(qh) @ np.abs(k[:, h]).T).max()))
    return out, weight, big


def attention_tol(out, weight, big):
    """The kernels sum in 32 bits and round the probabilities to fp16 (2^-11 of each, over values that are fp16 exactly
    or lie below its normal range, 2^-25) and the result once (2^-11 of it). A score is a sum of 128 products: off by
    128 * 2^-24 of their magnitude at most, the exponential by as much twice over (its own maximum, too)."""
    score = 2 * 128 * 2.0 ** -24 * big / np.sqrt(128.0)
    return np.abs(out) * 2.0 ** -11 + weight * (2.0 ** -11 + score + 2.0 ** -18) + 2.0 ** -24
