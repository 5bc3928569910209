// gfx950 kernels for the new tokens of a step, between a layer's QKV projection
// and its attention:
//
//   head_rows_kernel     heads of q and k normed and rotated; with a cache, k and v
//                        go into its pages (fp16, or E4M3 with one scale per tensor)
//   block_append_kernel  the same into a block-scaled E4M3 cache
//
// (No counterparts in the reference, whose caches take finished K and V.)
//
// A head's row is 128 fp16: 16 lanes hold 8 dims each, so a wave holds four rows
// and every load and store is 16 bytes a lane (8 for E4M3 codes). The norm's sum
// goes over the 16 lanes by rotations within them. A token's sines and cosines are
// computed once per wave or block, one pair a lane, and handed out through LDS:
// angles in 64 bits (position * frequency in half turns, less whole turns: the
// product of a position up to 2^31 is off by 2^-22 of a turn at most), sines of
// what is left in 32. No table of positions is read, and none limits them.

#include "pa_device.hpp"
#include "pa_fp8.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace pa {
namespace {

constexpr int kDims   = 8;                  // dims a lane holds of a row
constexpr int kLanes  = kHeadDim / kDims;   // lanes of a row
constexpr int kRows   = 64 / kLanes;        // rows of a wave
constexpr int kPairs  = kHeadDim / 2;       // most pairs of a rotation
constexpr int kMetaTable = 1, kMetaList = 2;
static_assert(kPairs == 64, "a wave computes one pair's sine and cosine per lane");

struct Turn {
    float c, s;
};

// Sum (or maximum) over the 16 lanes of a row, in every lane.
template <int CTRL>
__device__ __forceinline__ float rot16(float x) {
    const int v = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_sum(float x) {
    x += rot16<0x128>(x);
    x += rot16<0x124>(x);
    x += rot16<0x122>(x);
    return x + rot16<0x121>(x);
}
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, rot16<0x128>(x));
    x = fmaxf(x, rot16<0x124>(x));
    x = fmaxf(x, rot16<0x122>(x));
    return fmaxf(x, rot16<0x121>(x));
}

// Pair i's sine and cosine at a token (its `positions` row, or its place).
__device__ __forceinline__ Turn turn_of(const RopeTable& r, const int32_t* positions, int token, int place, int i) {
    const int pos = positions ? positions[static_cast<size_t>(token) * r.num_axes + r.axes[i]] : place;
    const double half = static_cast<double>(pos) * r.half_turns[i];
    const float  x    = static_cast<float>(half - 2.0 * rint(half * 0.5));   // [-1, 1]
    Turn t;
    sincospif(x, &t.s, &t.c);
    t.c *= r.scale;
    t.s *= r.scale;
    return t;
}

// What lane c of a row needs of a token's turns: interleaved pairs 4c .. 4c + 3
// (the first four), else pairs 8 (c mod h) .. + 7 with the sine's sign.
struct LaneTurns {
    Turn t[kDims];
};
__device__ __forceinline__ LaneTurns lane_turns(const RopeTable& r, const Turn* tab, int c) {
    LaneTurns l;
    const int  h = r.pairs / kDims;
    const bool upper = c >= h;
    if (r.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) l.t[e] = tab[min(4 * c + e, kPairs - 1)];
    } else {
        const int c0 = min(upper ? c - h : c, kLanes / 2 - 1);
#pragma unroll
        for (int e = 0; e < kDims; ++e) {
            l.t[e] = tab[kDims * c0 + e];
            if (!upper) l.t[e].s = -l.t[e].s;
        }
    }
    return l;
}

// A row chunk's 8 values normed (weight given) and turned, in 32 bits.
__device__ __forceinline__ void norm_turn(float (&y)[kDims], const HeadRows& rows, const RopeTable& r,
                                          const LaneTurns& l, int c) {
    if (rows.weight) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < kDims; ++e) sq = fmaf(y[e], y[e], sq);
        const float inv = 1.0f / sqrtf(row_sum(sq) * (1.0f / kHeadDim) + rows.eps);
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(rows.weight + kDims * c);
        const f32x4 w1 = *reinterpret_cast<const f32x4*>(rows.weight + kDims * c + 4);
#pragma unroll
        for (int e = 0; e < kDims; ++e) y[e] = y[e] * inv * (e < 4 ? w0[e & 3] : w1[e & 3]);
    }
    if (r.pairs == 0) return;
    const int  h      = r.pairs / kDims;   // lanes of one half
    const bool turned = c < 2 * h;
    if (r.interleaved) {
        if (turned) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = y[2 * e], b = y[2 * e + 1];
                y[2 * e]     = a * l.t[e].c - b * l.t[e].s;
                y[2 * e + 1] = b * l.t[e].c + a * l.t[e].s;
            }
        }
        return;
    }
    const int partner = (threadIdx.x & 63 & ~(kLanes - 1)) + (turned ? (c < h ? c + h : c - h) : c);
    float o[kDims];
#pragma unroll
    for (int e = 0; e < kDims; ++e) o[e] = __shfl(y[e], partner);
    if (turned) {
#pragma unroll
        for (int e = 0; e < kDims; ++e) y[e] = y[e] * l.t[e].c + o[e] * l.t[e].s;
    }
}

__device__ __forceinline__ void widen(float (&y)[kDims], const u32x4 x) {
#pragma unroll
    for (int e = 0; e < kDims; ++e) y[e] = f16_bits_to_f32((x[e >> 1] >> (16 * (e & 1))) & 0xffffu);
}
__device__ __forceinline__ u32x4 narrow(const float (&y)[kDims]) {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f16x2 h = {static_cast<_Float16>(y[2 * e]), static_cast<_Float16>(y[2 * e + 1])};
        o[e] = __builtin_bit_cast(uint32_t, h);
    }
    return o;
}

// Where a token goes. Every field is wave-uniform.
struct Place {
    bool ok;
    int  pos, page, slot;
};

// The entry that wave-uniform x belongs to: the last one with first(e) <= x, for
// first rising over n entries. `guess` is tried first (one round of loads).
template <class First>
__device__ __forceinline__ int entry_of(int x, int n, int guess, First first) {
    int lo = min(max(guess, 0), n - 1);
    if (first(lo) > x || (lo + 1 < n && first(lo + 1) <= x)) {
        lo = 0;
        int hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first(mid) <= x) lo = mid;
            else hi = mid;
        }
    }
    return lo;
}

// Entry e's page that holds the place pos (-1: none in range).
template <int META>
__device__ __forceinline__ int page_of(const RopeAppend& a, const int32_t* meta, int e, int pos) {
    if constexpr (META == kMetaList) {
        const int first = load_uniform(meta + a.n_ent, e);
        return load_uniform(meta + 3 * a.n_ent, load_uniform(meta + 2 * a.n_ent, e) + pos / a.page_size -
                                                    first / a.page_size);
    } else {
        const int row = a.slot_ids ? load_uniform(a.slot_ids, e) : e;
        const int i   = pos / a.page_size;
        if (pos < 0 || row < 0 || row >= a.table_rows || i >= a.table_stride) return -1;
        const int page = load_uniform(a.table + static_cast<size_t>(row) * a.table_stride, i);
        return page < a.num_pages ? page : -1;
    }
}

template <int META>
__device__ __forceinline__ Place place_of(const RopeAppend& a, const int32_t* meta, int t) {
    const int32_t* tok_begin = META == kMetaList ? meta : a.tok_begin;
    const int32_t* start     = META == kMetaList ? meta + a.n_ent : a.start;
    const int guess = static_cast<int>(static_cast<int64_t>(t) * a.n_ent / a.n_tok);
    const int e = entry_of(t, a.n_ent, guess, [&](int i) { return load_uniform(tok_begin, i); });
    Place p;
    const int st = load_uniform(start, e);
    p.pos  = static_cast<int>(static_cast<uint32_t>(st) +
                              static_cast<uint32_t>(t - load_uniform(tok_begin, e)));   // may wrap: then out of range
    p.page = st < 0 ? -1 : page_of<META>(a, meta, e, p.pos);
    p.ok   = p.page >= 0;
    p.slot = p.ok ? p.pos % a.page_size : 0;
    return p;
}

// The new table entries and lengths of a cache's append, spread over the grid.
__device__ __forceinline__ void write_tables(const RopeAppend& a, const int32_t* meta, int idx, int threads) {
    const int32_t* tab  = meta + 3 * a.n_ent + a.n_pl;
    const int32_t* lens = tab + 2 * a.n_tab;
    for (int i = idx; i < a.n_tab; i += threads) a.new_table[tab[2 * i]] = tab[2 * i + 1];
    for (int i = idx; i < a.n_len; i += threads) a.new_lens[lens[2 * i]] = lens[2 * i + 1];
}

// U groups of four rows of token t, from group g0 on: q's groups, then k's, then
// (with a cache) v's. CACHE: 0 none (k has an output), 1 fp16 pages, 2 E4M3 pages.
template <int CACHE, int META, int U>
__device__ __forceinline__ void rows_of_token(const RopeAppend& a, const int32_t* meta, int t, int g0, Turn* tab) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, r = lane / kLanes;
    const int gq = (a.q.heads + kRows - 1) / kRows, gk = (a.k.heads + kRows - 1) / kRows;
    const int groups = gq + gk + (CACHE ? gk : 0);
    u32x4 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int g = g0 + j;
        x[j] = u32x4{0, 0, 0, 0};
        if (g >= groups) continue;
        const bool q = g < gq, k = !q && g < gq + gk;
        const int  h = kRows * (q ? g : k ? g - gq : g - gq - gk) + r;
        const uint16_t* in = q ? a.q.in + t * a.q.in_stride : k ? a.k.in + t * a.k.in_stride : a.v + t * a.v_stride;
        if (h < (q ? a.q.heads : a.k.heads)) x[j] = load16<true>(in + h * kHeadDim + kDims * c);
    }
    Place p{true, 0, 0, 0};
    if constexpr (META != 0) p = place_of<META>(a, meta, t);
    LaneTurns l{};
    if (a.rope.pairs && g0 < gq + gk) {
        if (lane < a.rope.pairs) tab[lane] = turn_of(a.rope, a.positions, t, p.pos, lane);
        wave_lds_sync();
        l = lane_turns(a.rope, tab, c);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int g = g0 + j;
        if (g >= groups) continue;
        const bool q = g < gq, k = !q && g < gq + gk;
        const int  h = kRows * (q ? g : k ? g - gq : g - gq - gk) + r;
        float y[kDims];
        widen(y, x[j]);
        if (q || k) norm_turn(y, q ? a.q : a.k, a.rope, l, c);
        if (h >= (q ? a.q.heads : a.k.heads)) continue;
        if (q || CACHE == 0) {
            const HeadRows& rows = q ? a.q : a.k;
            __builtin_nontemporal_store(narrow(y), reinterpret_cast<u32x4*>(rows.out + t * rows.out_stride +
                                                                            h * kHeadDim + kDims * c));
            continue;
        }
        if constexpr (CACHE != 0) {
            if (!p.ok) continue;
            constexpr int EB = CACHE == 1 ? 2 : 1;
            unsigned char* dst = static_cast<unsigned char*>(k ? a.k_cache : a.v_cache) +
                                 kv_row_offset<EB>(p.page, h, p.slot, a.page_size, a.k.heads) + kDims * EB * c;
            if constexpr (CACHE == 1) {
                __builtin_nontemporal_store(k ? narrow(y) : x[j], reinterpret_cast<u32x4*>(dst));
            } else {
#pragma unroll
                for (int e = 0; e < kDims; ++e) y[e] *= k ? a.inv_k : a.inv_v;
                __builtin_nontemporal_store(e4m3_encode8(y), reinterpret_cast<u32x2*>(dst));
            }
        }
    }
}

constexpr int kRowWaves = 4;   // waves of a head_rows_kernel block, a token each

template <int CACHE, int META, int U>
__device__ __forceinline__ void head_rows_body(const RopeAppend& a, const int32_t* meta) {
    __shared__ Turn tab[kRowWaves][kPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t    = blockIdx.x * kRowWaves + wave;
    if constexpr (META == kMetaList)
        if (blockIdx.y == 0) write_tables(a, meta, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
    if (t >= a.n_tok) return;
    rows_of_token<CACHE, META, U>(a, meta, t, blockIdx.y * U, tab[wave]);
}

template <int CACHE, int META, int U>
__global__ __launch_bounds__(64 * kRowWaves) void head_rows_kernel(const RopeAppend a) {
    head_rows_body<CACHE, META, U>(a, a.meta);
}
// The meta is read where the arguments lie, as in pa_cache.hip.
template <int CACHE, int U, int N>
__global__ __launch_bounds__(64 * kRowWaves) void head_rows_inline_kernel(const RopeInline<N> x) {
    const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    head_rows_body<CACHE, kMetaList, U>(x.a, reinterpret_cast<const int32_t*>(args + offsetof(RopeInline<N>, meta)));
}

// ---- block-scaled caches ---------------------------------------------------

// The smallest k in [-32, 8] with amax <= 448 * 2^k (448 = 1.75 * 2^8).
__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    const int k = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(k, kBlockExpMin), kBlockExpMax);
}
__device__ __forceinline__ float exp2i(int k) { return __builtin_bit_cast(float, static_cast<uint32_t>(127 + k) << 23); }

__device__ __forceinline__ float wave_max(float x) {
    x = row_max(x);
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// One pool's part of a block: y holds the rows r + 4 i that lie in [s_lo, s_hi),
// zeros elsewhere. Returns the block's new exponent. `old`: the byte of the
// block's earlier rows (s_lo > 0).
__device__ __forceinline__ int store_block(float (&y)[4][kDims], unsigned char* rows, int old, int s_lo, int s_hi) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, r = lane / kLanes;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < kDims; ++e) amax = fmaxf(amax, fabsf(y[i][e]));
    int k = block_exponent(wave_max(amax));
    if (s_lo > 0) {
        const int before = old - 127;
        if (before >= k) {
            k = before;
        } else {
            // The earlier rows to the new scale. A NaN's byte stays as it is.
            const float f = exp2i(before - k);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r + 4 * i >= s_lo) continue;
                u32x2* at = reinterpret_cast<u32x2*>(rows + (r + 4 * i) * kHeadDim + kDims * c);
                const u32x2 was = *at;
                const f16x8 h   = fp8x8_to_f16x8(was[0], was[1]);
                float z[kDims];
#pragma unroll
                for (int e = 0; e < kDims; ++e) z[e] = static_cast<float>(h[e]) * f;
                u32x2 now = e4m3_encode8(z);
#pragma unroll
                for (int e = 0; e < kDims; ++e) {
                    const uint32_t m = 0xffu << (8 * (e & 3));
                    if (((was[e >> 2] >> (8 * (e & 3))) & 0x7fu) == 0x7fu)
                        now[e >> 2] = (now[e >> 2] & ~m) | (was[e >> 2] & m);
                }
                *at = now;
            }
        }
    }
    k = __builtin_amdgcn_readfirstlane(k);
    const float inv = exp2i(-k), top = k == kBlockExpMax ? kBlockTop : 448.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = r + 4 * i;
#pragma unroll
        for (int e = 0; e < kDims; ++e) y[i][e] *= inv;
        const u32x2 codes = e4m3_encode8(y[i], top);
        if (s >= s_lo && s < s_hi)
            __builtin_nontemporal_store(codes, reinterpret_cast<u32x2*>(rows + s * kHeadDim + kDims * c));
    }
    return k;
}

// One block of tokens of one entry, all its kv heads (a wave takes every
// waves-th); unit u counts them as the launch does: entry e's i-th block is unit
// tok_begin[e] / B + 2 e + i. (An entry of n tokens touches at most n / B + 2 blocks,
// so units of different entries never meet, whatever its start, which the host
// need not know.)
template <int META>
__device__ __forceinline__ void append_block(const RopeAppend& a, const int32_t* meta, int u, int waves,
                                             Turn (*tab)[kPairs]) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, r = lane / kLanes;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int B = a.block_tokens, P = a.page_size, hkv = a.k.heads;
    const int32_t* tok_begin = META == kMetaList ? meta : a.tok_begin;
    const int32_t* start     = META == kMetaList ? meta + a.n_ent : a.start;
    const int e = entry_of(u, a.n_ent, static_cast<int>(static_cast<int64_t>(u) * a.n_ent / a.units),
                           [&](int i) { return load_uniform(tok_begin, i) / B + 2 * i; });
    const int t0 = load_uniform(tok_begin, e), st = load_uniform(start, e);
    const int t1 = META == kMetaList && e + 1 == a.n_ent ? a.n_tok : min(load_uniform(tok_begin, e + 1), a.n_tok);
    if (st < 0 || t0 < 0 || t1 <= t0 || st > INT_MAX - (t1 - t0) - B) return;
    const int blk = st / B + (u - (t0 / B + 2 * e));   // block of the sequence
    const int lo = max(st, blk * B), hi = min(st + (t1 - t0), (blk + 1) * B);
    if (lo >= hi) return;
    const int page = page_of<META>(a, meta, e, lo);
    if (page < 0) return;
    const int s_lo = lo - blk * B, s_hi = hi - blk * B;
    const int tok  = t0 + (lo - st);          // token at s_lo
    const int b    = blk * B % P / B;         // block of the page
    if (a.rope.pairs) {
        const int threads = 64 * waves;
        for (int i = threadIdx.x; i < (s_hi - s_lo) * kPairs; i += threads) {
            const int s = s_lo + i / kPairs, p = i % kPairs;
            if (p < a.rope.pairs) tab[s][p] = turn_of(a.rope, a.positions, tok + s - s_lo, blk * B + s, p);
        }
        __syncthreads();
    }
    for (int h = wave; h < hkv; h += waves) {
        u32x4 kx[4], vx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = r + 4 * i;
            kx[i] = vx[i] = u32x4{0, 0, 0, 0};
            if (s >= s_lo && s < s_hi) {
                const size_t t = static_cast<size_t>(tok + s - s_lo);
                kx[i] = load16<true>(a.k.in + t * a.k.in_stride + h * kHeadDim + kDims * c);
                vx[i] = load16<true>(a.v + t * a.v_stride + h * kHeadDim + kDims * c);
            }
        }
        uint16_t* sc = reinterpret_cast<uint16_t*>(a.scales) + (static_cast<size_t>(page) * hkv + h) * (P / B) + b;
        const int old = s_lo > 0 ? *sc : 0;
        const size_t row0 = kv_row_offset<1>(page, h, b * B, P, hkv);
        float y[4][kDims];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            widen(y[i], kx[i]);
            LaneTurns l{};
            if (a.rope.pairs) l = lane_turns(a.rope, tab[min(r + 4 * i, 15)], c);
            norm_turn(y[i], a.k, a.rope, l, c);
            const int s = r + 4 * i;
            if (s < s_lo || s >= s_hi) {
#pragma unroll
                for (int e2 = 0; e2 < kDims; ++e2) y[i][e2] = 0.f;
            }
        }
        const int kk = store_block(y, static_cast<unsigned char*>(a.k_cache) + row0, old & 0xff, s_lo, s_hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) widen(y[i], vx[i]);
        const int kv = store_block(y, static_cast<unsigned char*>(a.v_cache) + row0, old >> 8, s_lo, s_hi);
        if (lane == 0) *sc = static_cast<uint16_t>((kk + 127) | ((kv + 127) << 8));
    }
}

// Blocks of the grid: the units of k and v, then the tokens' q rows.
template <int META>
__device__ __forceinline__ void block_append_body(const RopeAppend& a, const int32_t* meta) {
    __shared__ Turn tab[16][kPairs];
    const int waves = blockDim.x >> 6;
    if constexpr (META == kMetaList)
        write_tables(a, meta, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
    if (static_cast<int>(blockIdx.x) < a.units) {
        append_block<META>(a, meta, blockIdx.x, waves, tab);
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int gq = (a.q.heads + kRows - 1) / kRows;
    const int w  = (blockIdx.x - a.units) * waves + wave;
    const int t  = w / gq;
    if (t >= a.n_tok) return;
    RopeAppend q = a;
    q.k.heads = 0;
    rows_of_token<0, META, 1>(q, meta, t, w - t * gq, tab[wave]);
}

constexpr int kBlockWaves = 8;

template <int META>
__global__ __launch_bounds__(64 * kBlockWaves) void block_append_kernel(const RopeAppend a) {
    block_append_body<META>(a, a.meta);
}
template <int N>
__global__ __launch_bounds__(64 * kBlockWaves) void block_append_inline_kernel(const RopeInline<N> x) {
    const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    block_append_body<kMetaList>(x.a, reinterpret_cast<const int32_t*>(args + offsetof(RopeInline<N>, meta)));
}

int groups_of(const RopeAppend& a, bool cache) {
    const int gq = (a.q.heads + kRows - 1) / kRows, gk = (a.k.heads + kRows - 1) / kRows;
    return gq + gk + (cache ? gk : 0);
}

template <int CACHE, int META>
void launch_rows(const RopeAppend& a, hipStream_t s) {
    const dim3 grid((a.n_tok + kRowWaves - 1) / kRowWaves, groups_of(a, CACHE != 0));
    hipLaunchKernelGGL((head_rows_kernel<CACHE, META, 1>), grid, dim3(64 * kRowWaves), 0, s, a);
}
template <int CACHE, int N>
void launch_rows_inline(const RopeAppend& a, const int32_t* meta, size_t n, hipStream_t s) {
    RopeInline<N> x;
    x.a = a;
    std::copy(meta, meta + n, x.meta);
    const dim3 grid((a.n_tok + kRowWaves - 1) / kRowWaves, groups_of(a, CACHE != 0));
    hipLaunchKernelGGL((head_rows_inline_kernel<CACHE, 1, N>), grid, dim3(64 * kRowWaves), 0, s, x);
}

// Waves of a block and blocks of a block_append_kernel launch; sets a.units.
dim3 block_grid(RopeAppend& a, int& waves) {
    waves = std::min(a.k.heads, kBlockWaves);
    a.block_tokens = block_tokens(a.page_size);
    a.units = a.n_tok / a.block_tokens + 2 * a.n_ent;
    const long q = static_cast<long>(a.n_tok) * ((a.q.heads + kRows - 1) / kRows);
    return dim3(static_cast<unsigned>(a.units + (q + waves - 1) / waves));
}
template <int N>
void launch_block_inline(RopeAppend a, const int32_t* meta, size_t n, hipStream_t s) {
    int waves = 0;
    const dim3 grid = block_grid(a, waves);
    RopeInline<N> x;
    x.a = a;
    std::copy(meta, meta + n, x.meta);
    hipLaunchKernelGGL((block_append_inline_kernel<N>), grid, dim3(64 * waves), 0, s, x);
}

}  // namespace

hipError_t launch_norm_rope(const RopeAppend& a, hipStream_t s) {
    if (a.n_tok <= 0 || groups_of(a, false) == 0) return hipSuccess;
    launch_rows<0, 0>(a, s);
    return hipGetLastError();
}

hipError_t launch_append_rope(int dtype, const RopeAppend& a, const int32_t* meta, size_t n_meta, hipStream_t s) {
    check_kv_dtype(dtype);
    if (a.n_tok <= 0) return hipSuccess;
    const bool list = meta || a.meta;   // a cache's append; else the caller's device arrays
    if (dtype == PA_KV_FP8_E4M3_BLOCK) {
        if (meta && n_meta <= 256) {
            launch_block_inline<256>(a, meta, n_meta, s);
        } else if (meta) {
            launch_block_inline<kRopeInlineInts>(a, meta, n_meta, s);
        } else {
            RopeAppend b = a;
            int waves = 0;
            const dim3 grid = block_grid(b, waves);
            if (list) hipLaunchKernelGGL(block_append_kernel<kMetaList>, grid, dim3(64 * waves), 0, s, b);
            else hipLaunchKernelGGL(block_append_kernel<kMetaTable>, grid, dim3(64 * waves), 0, s, b);
        }
        return hipGetLastError();
    }
    const bool fp16 = dtype == PA_KV_FP16;
    if (meta && n_meta <= 256) {
        if (fp16) launch_rows_inline<1, 256>(a, meta, n_meta, s);
        else launch_rows_inline<2, 256>(a, meta, n_meta, s);
    } else if (meta) {
        if (fp16) launch_rows_inline<1, kRopeInlineInts>(a, meta, n_meta, s);
        else launch_rows_inline<2, kRopeInlineInts>(a, meta, n_meta, s);
    } else if (list) {
        if (fp16) launch_rows<1, kMetaList>(a, s);
        else launch_rows<2, kMetaList>(a, s);
    } else {
        if (fp16) launch_rows<1, kMetaTable>(a, s);
        else launch_rows<2, kMetaTable>(a, s);
    }
    return hipGetLastError();
}

}  // namespace pa
