// gfx950 kernels for the new tokens of a step, between a layer's QKV projection
// and its attention:
//
//   head_rows_kernel     heads of q and k normed and rotated; with a cache, k and v
//                        go into its pages (fp16, or E4M3 with one scale per tensor)
//   block_append_kernel  the same into a block-scaled E4M3 cache
//
// (No counterparts in the reference, whose caches take finished K and V.)
//
//   y = x w / sqrt(mean(x^2) + eps); (a, b) -> s (a cos t - b sin t, b cos t + a sin t)
//
// with t = position * frequency of the pair, in 32 bits, rounded once.
//
// A head's row is 128 fp16: 16 lanes hold 8 dims each, a wave four rows. The norm's
// sum goes over the 16 lanes by rotations within them. A token's sines and cosines are
// computed once per wave or block, one pair a lane, and handed out through LDS:
// angles in 64 bits (position * frequency in half turns, less whole turns: the
// product of a position up to 2^31 is off by 2^-22 of a turn at most), sines of
// what is left in 32. No table of positions is read, and none limits them.
//
// Bound by memory from some thousand tokens on: 8192 tokens of 32 + 8 heads take 30 us
// (168 MB, 5.6 TB/s; a copy of as many bytes 33), of which the arithmetic is half
// (SQ_ACTIVE_INST_VALU), 8 x 4096 tokens of 32 + 2 x 8 into block-scaled pages 133
// us (738 MB, 5.5 TB/s); below by the chain kernel arguments, entry, place, rows,
// store: 2.4 us for one token, 3.1 for a step of 64 into fp16 pages, 4.2 into
// block-scaled ones.

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
constexpr int kStoreAux = 2;   // buffer stores are non-temporal: what is stored is read by later kernels only
// ... and loads where NT is given: see streams().
template <bool NT> constexpr int kLoadAux = NT ? 2 : 0;

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

// What turns pair i, loaded before a wave looks up its token's place: the lookup's
// loads would otherwise be waited for first. (Into block-scaled pages: a step of 64
// sequences 4.3 -> 4.2 us, a prompt of 333 tokens 6.7 -> 6.3.)
struct Pair {
    double half_turns;   // per position
    int    axis;
};
__device__ __forceinline__ Pair pair_of(const RopeTable& r, int i) {
    Pair p{0.0, 0};
    if (i < r.pairs) {
        p.half_turns = r.half_turns[i];
        if (r.num_axes > 1) p.axis = r.axes[i];
    }
    return p;
}
// Its sine and cosine at a token (its `positions` row, or its place).
__device__ __forceinline__ Turn turn_of(const RopeTable& r, const Pair& p, const int32_t* positions, int token,
                                        int place) {
    const int    pos  = positions ? positions[static_cast<size_t>(token) * r.num_axes + p.axis] : place;
    const double half = static_cast<double>(pos) * p.half_turns;
    const float  x    = static_cast<float>(half - 2.0 * rint(half * 0.5));   // [-1, 1]
    Turn t;
    sincospif(x, &t.s, &t.c);
    t.c *= r.scale;
    t.s *= r.scale;
    return t;
}

// The 8 dims that lane c of a row holds, as two chunks of four: with half-split
// pairs both halves of pairs 4c .. 4c + 3, so that no lane needs another's values
// (the dims that do not turn are halved likewise: a load then takes runs of whole
// 64 bytes); with interleaved ones, eight dims in a row.
struct LaneDims {
    int  lo, hi;   // the chunks' first dims
    bool turned;
};
template <bool INTER>
__device__ __forceinline__ LaneDims lane_dims(int pairs, int c) {
    const bool turned = 4 * c < pairs;
    if constexpr (INTER) return {kDims * c, kDims * c + 4, turned};
    const int lo = 4 * c + (turned ? 0 : pairs);   // 2 * pairs + 4 (c - pairs / 4)
    return {lo, lo + (turned ? pairs : kPairs - pairs), turned};
}

// A lane's dims of the row `off` bytes into a resource (past its end: zeros).
template <bool INTER, bool NT>
__device__ __forceinline__ u32x4 load_dims(__amdgpu_buffer_rsrc_t rs, const LaneDims& d, int off) {
    if constexpr (INTER)
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 2 * d.lo + off, 0, kLoadAux<NT>));
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, 2 * d.lo + off, 0, kLoadAux<NT>));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, 2 * d.hi + off, 0, kLoadAux<NT>));
    return u32x4{x[0], x[1], y[0], y[1]};
}
// The same stored, as fp16 or as codes (past the end: dropped).
template <bool INTER>
__device__ __forceinline__ void store_dims(__amdgpu_buffer_rsrc_t rs, const LaneDims& d, int off, u32x4 x) {
    if constexpr (INTER) return __builtin_amdgcn_raw_buffer_store_b128(x, rs, 2 * d.lo + off, 0, kStoreAux);
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{x[0], x[1]}, rs, 2 * d.lo + off, 0, kStoreAux);
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{x[2], x[3]}, rs, 2 * d.hi + off, 0, kStoreAux);
}
template <bool INTER>
__device__ __forceinline__ void store_dims(__amdgpu_buffer_rsrc_t rs, const LaneDims& d, int off, u32x2 x) {
    if constexpr (INTER) return __builtin_amdgcn_raw_buffer_store_b64(x, rs, d.lo + off, 0, kStoreAux);
    __builtin_amdgcn_raw_buffer_store_b32(x[0], rs, d.lo + off, 0, kStoreAux);
    __builtin_amdgcn_raw_buffer_store_b32(x[1], rs, d.hi + off, 0, kStoreAux);
}

// A row's norm weights, and a token's turns, as a lane needs them.
struct LaneWeights {
    f32x4 w[2];
};
struct LaneTurns {
    Turn t[4];
};
__device__ __forceinline__ LaneWeights lane_weights(const float* weight, const LaneDims& d) {
    if (!weight) return {};
    return {{*reinterpret_cast<const f32x4*>(weight + d.lo), *reinterpret_cast<const f32x4*>(weight + d.hi)}};
}
__device__ __forceinline__ LaneTurns lane_turns(const Turn* tab, int c) {
    LaneTurns l;
#pragma unroll
    for (int e = 0; e < 4; ++e) l.t[e] = tab[4 * c + e];
    return l;
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

// 1 / sqrt(mean of a row's squares + eps). (v_rsq_f32 is off by 2^-23 at most. Its
// input is no fp32 subnormal, which it would flush: the mean of squares of fp16
// values is 0 or at least 2^-55.)
__device__ __forceinline__ float inv_norm(const float (&y)[kDims], float eps) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < kDims; ++e) sq = fmaf(y[e], y[e], sq);
    return __builtin_amdgcn_rsqf(fmaf(row_sum(sq), 1.0f / kHeadDim, eps));
}

// A lane's 8 values of a row under their norm (inv: the row's inv_norm), and turned.
__device__ __forceinline__ void apply_norm(float (&y)[kDims], float inv, const LaneWeights& w) {
#pragma unroll
    for (int e = 0; e < kDims; ++e) y[e] = y[e] * inv * w.w[e / 4][e % 4];
}
template <bool INTER>
__device__ __forceinline__ void apply_turns(float (&y)[kDims], const LaneTurns& l) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : 4 + e;
        const float a = y[i], b = y[j];
        y[i] = a * l.t[e].c - b * l.t[e].s;
        y[j] = b * l.t[e].c + a * l.t[e].s;
    }
}

// Where a token goes. Every field is wave-uniform.
struct Place {
    bool ok;
    int  pos, page, slot;
};

// The entry that wave-uniform x belongs to: the last one with first(i) <= x, for
// first rising over n entries. `guess` is tried first (scalar loads, one round);
// else each round has every lane look at one of 64 evenly spaced entries. (With a
// binary search's scalar loads, one after the other, 64 sequences' step into a
// block-scaled cache took 1 us more.)
template <class First, class FirstOf>
__device__ __forceinline__ int entry_of(int x, int n, int guess, First first, FirstOf first_of) {
    int lo = min(max(guess, 0), n - 1);
    if (first(lo) <= x && (lo + 1 >= n || first(lo + 1) > x)) return lo;
    lo = 0;
    for (int span = n; span > 1;) {   // it is one of lo .. lo + span - 1
        const int step = (span + 63) / 64;
        const int i    = lo + step * static_cast<int>(threadIdx.x & 63);
        const bool le  = i < lo + span && first_of(i) <= x;
        // Rising: the lanes that hold are the first ones (lane 0 among them, unless none is).
        const int at = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(le)) - 1, 0);
        const int end = lo + span;
        lo += step * at;
        span = min(step, end - lo);
    }
    return lo;
}

// Entry e's page that holds the place pos (-1: none in range).
template <int META>
__device__ __forceinline__ int page_of(const RopeAppend& a, const int32_t* meta, int e, int pos) {
    if constexpr (META == kMetaList) {
        const int first = load_uniform(meta + a.n_ent, e);
        return load_uniform(meta + 3 * a.n_ent, load_uniform(meta + 2 * a.n_ent, e) + a.by_page.page(pos) -
                                                    a.by_page.page(first));
    } else {
        const int row = a.slot_ids ? load_uniform(a.slot_ids, e) : e;
        const int i   = a.by_page.page(pos);   // below 0: refused with the place
        if (pos < 0 || row < 0 || row >= a.table_rows || i >= a.table_stride) return -1;
        const int page = load_uniform(a.table + static_cast<size_t>(row) * a.table_stride, i);
        return page < a.num_pages ? page : -1;
    }
}

template <int META>
__device__ __forceinline__ Place place_of(const RopeAppend& a, const int32_t* meta, int t) {
    const int32_t* tok_begin = META == kMetaList ? meta : a.tok_begin;
    const int32_t* start     = META == kMetaList ? meta + a.n_ent : a.start;
    const int guess = static_cast<int>(static_cast<float>(t) * a.ent_rate);
    const int e = entry_of(
        t, a.n_ent, guess, [&](int i) { return load_uniform(tok_begin, i); }, [&](int i) { return tok_begin[i]; });
    Place p;
    const int st = load_uniform(start, e), t0 = load_uniform(tok_begin, e);
    p.pos = static_cast<int>(static_cast<uint32_t>(st) + static_cast<uint32_t>(t - t0));   // may wrap: then out of range
    // A caller's arrays may leave tokens out on both sides (a padded batch's).
    const bool none = META == kMetaTable && (st < 0 || t < t0 || t >= load_uniform(tok_begin, e + 1));
    p.page = none ? -1 : page_of<META>(a, meta, e, p.pos);
    p.ok   = p.page >= 0;
    p.slot = p.ok ? p.pos - a.by_page.page(p.pos) * a.page_size : 0;
    return p;
}

// The new table entries and lengths of a cache's append, spread over the grid.
__device__ __forceinline__ void write_tables(const RopeAppend& a, const int32_t* meta, int idx, int threads) {
    const int32_t* tab  = meta + 3 * a.n_ent + a.n_pl;
    const int32_t* lens = tab + 2 * a.n_tab;
    for (int i = idx; i < a.n_tab; i += threads) a.new_table[tab[2 * i]] = tab[2 * i + 1];
    for (int i = idx; i < a.n_len; i += threads) a.new_lens[lens[2 * i]] = lens[2 * i + 1];
}

// What a wave's groups of four rows are.
enum RowKind { kRowQ = 0, kRowK = 1, kRowV = 2 };

// Up to U groups of four rows of one kind of token t, from group g0 on. CACHE: 0
// none (k has an output), 1 fp16 pages, 2 E4M3 pages. All loads go out first; the
// token's place and turns are worked out under them. Loads and stores go through
// buffer resources that end with the token's heads, so a group with fewer than
// four rows, or none, takes no branch (branches around the loads had the compiler
// wait for each group's before the next: 8192 tokens of 32 + 8 heads 32.8 us at 8
// groups a wave, but 37.1 at 4 and 66.8 at 6).
template <int CACHE, bool INTER, int META, int U, bool NT>
__device__ __forceinline__ void rows_of_token(const RopeAppend& a, const int32_t* meta, int t, int kind, int g0,
                                              Turn* tab) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, r = lane / kLanes;
    const bool v = CACHE != 0 && kind == kRowV;
    const HeadRows& rows = kind == kRowQ ? a.q : a.k;
    const int heads = rows.heads, h0 = kRows * g0;
    const LaneDims d = lane_dims<INTER>(v ? 0 : a.rope.pairs, c);
    const Pair pair = pair_of(a.rope, v ? kPairs : lane);
    const uint16_t* in = (v ? a.v + t * a.v_stride : rows.in + t * rows.in_stride) + h0 * kHeadDim;
    const __amdgpu_buffer_rsrc_t src = buffer_rsrc(in, 2 * kHeadDim * (heads - h0));
    u32x4 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = load_dims<INTER, NT>(src, d, 2 * kHeadDim * (kRows * j + r));
    Place p{true, 0, 0, 0};
    if constexpr (META != 0) p = place_of<META>(a, meta, t);
    const bool norm = !v && rows.weight != nullptr;
    const LaneWeights w = lane_weights(v ? nullptr : rows.weight, d);
    LaneTurns l{};
    if (!v && a.rope.pairs) {
        if (lane < a.rope.pairs) tab[lane] = turn_of(a.rope, pair, a.positions, t, p.pos);
        wave_lds_sync();
        l = lane_turns(tab, c);
    }
    auto finish = [&](float (&y)[kDims]) {
        if (norm) apply_norm(y, inv_norm(y, rows.eps), w);
        if (d.turned) apply_turns<INTER>(y, l);
    };
    if (CACHE == 0 || kind == kRowQ) {
        uint16_t* out = rows.out + t * rows.out_stride + h0 * kHeadDim;
        const __amdgpu_buffer_rsrc_t dst = buffer_rsrc(out, 2 * kHeadDim * (heads - h0));
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (h0 + kRows * j >= heads) break;
            float y[kDims];
            widen(y, x[j]);
            finish(y);
            store_dims<INTER>(dst, d, 2 * kHeadDim * (kRows * j + r), narrow(y));
        }
        return;
    }
    if constexpr (CACHE != 0) {
        if (!p.ok) return;
        constexpr int EB = CACHE == 1 ? 2 : 1;
        const int head_bytes = a.page_size * kRowBytes<EB>;   // a page's bytes fit 31 bits
        unsigned char* page = static_cast<unsigned char*>(v ? a.v_cache : a.k_cache) +
                              static_cast<size_t>(p.page) * heads * head_bytes + static_cast<size_t>(h0) * head_bytes;
        const __amdgpu_buffer_rsrc_t dst = buffer_rsrc(page, (heads - h0) * head_bytes);
        const int slot = p.slot * kRowBytes<EB>;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (h0 + kRows * j >= heads) break;
            // (A row without a head goes past the end by name: its offset may reach 2^32.)
            const int row = kRows * j + r;
            const int off = h0 + row < heads ? row * head_bytes + slot : INT_MIN;
            float y[kDims];
            widen(y, x[j]);
            finish(y);
            if constexpr (CACHE == 1) {
                store_dims<INTER>(dst, d, off, v ? x[j] : narrow(y));
            } else {
                const float inv = v ? a.inv_v : a.inv_k;
#pragma unroll
                for (int e = 0; e < kDims; ++e) y[e] *= inv;
                store_dims<INTER>(dst, d, off, e4m3_encode8(y));
            }
        }
    }
}

constexpr int kRowWaves = 4;   // waves of a head_rows_kernel block

// Wave w takes part w % (pq + pk [+ pk]) of a token: U groups of q, of k, or of v.
template <int CACHE, bool INTER, int META, int U, bool NT>
__device__ __forceinline__ void head_rows_body(const RopeAppend& a, const int32_t* meta) {
    __shared__ __attribute__((aligned(16))) Turn tab[kRowWaves][kPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w    = blockIdx.x * kRowWaves + wave;
    const int t    = a.by_parts.page(w);
    if constexpr (META == kMetaList)
        write_tables(a, meta, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
    if (t >= a.n_tok) return;
    int part = w - t * a.parts, kind = kRowQ;
    if (part >= a.parts_q) {
        part -= a.parts_q;
        kind = kRowK;
        if (CACHE != 0 && part >= a.parts_k) {
            part -= a.parts_k;
            kind = kRowV;
        }
    }
    rows_of_token<CACHE, INTER, META, U, NT>(a, meta, t, kind, part * U, tab[wave]);
}

template <int CACHE, bool INTER, int META, int U, bool NT>
__global__ __launch_bounds__(64 * kRowWaves) void head_rows_kernel(const RopeAppend a) {
    head_rows_body<CACHE, INTER, META, U, NT>(a, a.meta);
}
// The meta is read where the arguments lie, as in pa_cache.hip. (Calls that fit there
// are short, but for prompts into pages of 64 tokens and more: those never take the
// streaming loads, which would save them 2 to 5%.)
template <int CACHE, bool INTER, int U, int N>
__global__ __launch_bounds__(64 * kRowWaves) void head_rows_inline_kernel(const RopeInline<N> x) {
    const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    head_rows_body<CACHE, INTER, kMetaList, U, false>(
        x.a, reinterpret_cast<const int32_t*>(args + offsetof(RopeInline<N>, meta)));
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

// One block of tokens of one entry in one pool (its keys, or its values), a wave for
// each of the kv heads from h0 on. Unit u counts blocks as the launch does:
// entry e's i-th block is unit tok_begin[e] / B + 2 e + i. (An entry of n tokens
// touches at most n / B + 2 blocks, so units of different entries never meet,
// whatever its start, which the host need not know.) Where that makes more units
// than tokens, as in a decode step, a unit is a token, and the first of a block takes it.
//
// A wave holds the block's 16 rows of a head as they came (four a load, as in the
// rows kernel), norms and turns them once for their largest magnitude and, with the
// scale that it asks for, once more for the codes: 160 more instructions a wave, but
// half the registers, and so twice the waves, of holding the results (8 x 4096
// tokens 166 us with keys and values in one wave and 145 registers, 150 with values
// worked out twice and 112, 138.5 with 89 for one head a wave). The codes of
// earlier rows and their scale are loaded beside the new rows: a scale grows in some
// 2% of a decode step's blocks, so in nearly every step, and would cost it a further
// trip to memory (where none grows the loads cost 0.1 us at 64 sequences, 0.5 at 512).
template <bool INTER, int META, bool V, bool NT>
__device__ __forceinline__ void append_block(const RopeAppend& a, const int32_t* meta, int u, int h0, int waves,
                                             Turn (*tab)[kPairs]) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, r = lane / kLanes;
    const int h = h0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = a.block_shift, B = 1 << sh, P = a.page_size, hkv = a.k.heads;
    const int32_t* tok_begin = META == kMetaList ? meta : a.tok_begin;
    const int32_t* start     = META == kMetaList ? meta + a.n_ent : a.start;
    const Pair pair = pair_of(a.rope, V ? kPairs : lane);   // the thread's: it takes every waves-th token's
    const bool by_token = a.by_token != 0;
    const int  div = by_token ? 0 : sh, plus = by_token ? 0 : 2;
    const int  guess = static_cast<int>(fmaf(static_cast<float>(u), a.ent_rate, 0.5f));
    const int e = entry_of(
        u, a.n_ent, guess, [&](int i) { return (load_uniform(tok_begin, i) >> div) + plus * i; },
        [&](int i) { return (tok_begin[i] >> div) + plus * i; });
    const int t0 = load_uniform(tok_begin, e), st = load_uniform(start, e);
    const int t1 = META == kMetaList && e + 1 == a.n_ent ? a.n_tok : min(load_uniform(tok_begin, e + 1), a.n_tok);
    if (st < 0 || t0 < 0 || t1 <= t0 || st > INT_MAX - (t1 - t0) - B) return;
    if (u < (t0 >> div) + plus * e) return;   // a token before the first entry
    // Block of the sequence. (One that an earlier token of the entry lies in has its unit there.)
    if (by_token && u > t0 && ((st + (u - t0)) & (B - 1)) != 0) return;
    const int blk = by_token ? (st + (u - t0)) >> sh : (st >> sh) + (u - ((t0 >> sh) + 2 * e));
    const int lo = max(st, blk * B), hi = min(st + (t1 - t0), (blk + 1) * B);
    if (lo >= hi) return;
    const int s_lo = lo - blk * B, s_hi = hi - blk * B;
    const int tok  = t0 + (lo - st);          // token at s_lo
    const LaneDims d = lane_dims<INTER || V>(V ? 0 : a.rope.pairs, c);
    // The new rows, on their way under the page's lookup and the turns. Rows outside
    // the block's part of the entry read zeros. (Strides are below 2^26.)
    const long stride = V ? a.v_stride : a.k.in_stride;
    const __amdgpu_buffer_rsrc_t src = buffer_rsrc((V ? a.v : a.k.in) + tok * stride, h < hkv ? INT_MAX : 0);
    u32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = r + kRows * i;
        const int off = s >= s_lo && s < s_hi ? 2 * ((s - s_lo) * static_cast<int>(stride) + h * kHeadDim) : INT_MIN;
        x[i] = load_dims<INTER || V, NT>(src, d, off);
    }
    const int page = page_of<META>(a, meta, e, lo);
    if (!V && a.rope.pairs) {
        for (int s = s_lo + (threadIdx.x >> 6); s < s_hi; s += waves)
            if (lane < a.rope.pairs) tab[s][lane] = turn_of(a.rope, pair, a.positions, tok + s - s_lo, blk * B + s);
    }
    if (page < 0) return;
    const bool norm = !V && a.k.weight != nullptr;
    const LaneWeights w = lane_weights(V ? nullptr : a.k.weight, d);
    // The head's earlier rows (none past s_lo is read) and their scale.
    const int b = (blk * B - a.by_page.page(blk * B) * P) >> sh;   // block of the page
    uint8_t* const sc = a.scales + 2 * ((static_cast<size_t>(page) * hkv + h) * (P >> sh) + b) + (V ? 1 : 0);
    unsigned char* const rows = static_cast<unsigned char*>(V ? a.v_cache : a.k_cache) + kv_row_offset<1>(page, h, b * B, P, hkv);
    const bool earlier = s_lo > 0 && h < hkv;
    const __amdgpu_buffer_rsrc_t held = buffer_rsrc(rows, earlier ? s_lo * kHeadDim : 0);
    const int old = earlier ? *sc : 0;
    u32x2 was[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        was[i] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_raw_buffer_load_b64(held, (r + kRows * i) * kHeadDim + kDims * c, 0, 0));
    if (!V && a.rope.pairs) __syncthreads();
    if (h >= hkv) return;
    float amax = 0.f, inv_n[4];
    auto value = [&](float (&y)[kDims], int i) {   // row r + 4 i, its norm known
        if (norm) apply_norm(y, inv_n[i], w);
        if (!V && d.turned) apply_turns<INTER>(y, lane_turns(tab[r + kRows * i], c));
    };
    // Four rows at a time, those that hold none of the new tokens left out.
    auto live = [&](int i) { return s_lo < kRows * (i + 1) && kRows * i < s_hi; };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        inv_n[i] = 1.0f;
        if (!live(i)) continue;
        float y[kDims];
        widen(y, x[i]);
        inv_n[i] = norm ? inv_norm(y, a.k.eps) : 1.0f;
        value(y, i);
        float m = 0.f;
#pragma unroll
        for (int n = 0; n < kDims; ++n) m = fmaxf(m, fabsf(y[n]));
        const int s = r + kRows * i;
        if (s >= s_lo && s < s_hi) amax = fmaxf(amax, m);
        // The second time through starts from the rows again: the compiler would keep y.
        asm volatile("" : "+v"(x[i]), "+v"(inv_n[i])::"memory");
    }
    int k = __builtin_amdgcn_readfirstlane(block_exponent(wave_max(amax)));
    if (s_lo > 0) {
        const int before = __builtin_amdgcn_readfirstlane(old) - 127;
        if (before < k) {
            // The earlier rows to the new scale. A NaN's byte stays as it is.
            const float f = exp2i(max(before - k, -126));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f16x8 g = fp8x8_to_f16x8(was[i][0], was[i][1]);
                float z[kDims];
#pragma unroll
                for (int n = 0; n < kDims; ++n) z[n] = static_cast<float>(g[n]) * f;
                u32x2 now = e4m3_encode8(z);
#pragma unroll
                for (int n = 0; n < kDims; ++n) {
                    const uint32_t m = 0xffu << (8 * (n & 3));
                    if (((was[i][n >> 2] >> (8 * (n & 3))) & 0x7fu) == 0x7fu)
                        now[n >> 2] = (now[n >> 2] & ~m) | (was[i][n >> 2] & m);
                }
                __builtin_amdgcn_raw_buffer_store_b64(now, held, (r + kRows * i) * kHeadDim + kDims * c, 0, 0);
                asm volatile("" ::: "memory");
            }
        }
        k = max(k, before);
    }
    const float inv = exp2i(-k), top = k == kBlockExpMax ? kBlockTop : 448.0f;
    const __amdgpu_buffer_rsrc_t dst = buffer_rsrc(rows, s_hi * kHeadDim);   // no row past the new ones is written
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!live(i)) continue;
        const int s = r + kRows * i;
        float y[kDims];
        widen(y, x[i]);
        value(y, i);
#pragma unroll
        for (int n = 0; n < kDims; ++n) y[n] *= inv;
        const u32x2 codes = e4m3_encode8(y, top);
        if (s >= s_lo) store_dims<INTER || V>(dst, d, s * kHeadDim, codes);
        asm volatile("" ::: "memory");
    }
    if (lane == 0) *sc = static_cast<uint8_t>(k + 127);
}

// Groups of a token's q rows that one wave takes beside the blocks.
constexpr int kBlockQ = 4;

// Blocks of the grid: the units of k and v in turn (a streaming call's, which is long
// enough to have both at once anyway, k before v), then the tokens' q rows. us with
// k before v and in turn: 37 ragged prompts 24.1 / 22.8, 4096 tokens 18.5 / 18.3,
// 64 single tokens 4.3 / 4.3, 8 x 4096 tokens 133.9 / 137.2; q first 24.6, 19.8, 4.5,
// 133.4.
template <bool INTER, int META, bool NT>
__device__ __forceinline__ void block_append_body(const RopeAppend& a, const int32_t* meta) {
    __shared__ __attribute__((aligned(16))) Turn tab[16][kPairs];
    const int waves = blockDim.x >> 6;
    if constexpr (META == kMetaList)
        write_tables(a, meta, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
    const int blocks = a.units * a.head_groups;   // of k, and of v
    if (static_cast<int>(blockIdx.x) < 2 * blocks) {
        const int  n = blockIdx.x;
        const bool v = NT ? n >= blocks : (n & 1) != 0;
        const int  i = NT ? n - (v ? blocks : 0) : n >> 1;
        const int  u = a.head_groups == 1 ? i : i / a.head_groups, h0 = (i - u * a.head_groups) * waves;
        if (v) append_block<INTER, META, true, NT>(a, meta, u, h0, waves, tab);
        else append_block<INTER, META, false, NT>(a, meta, u, h0, waves, tab);
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = (blockIdx.x - 2 * blocks) * waves + wave;
    const int t = a.by_parts.page(w);
    if (t >= a.n_tok) return;
    rows_of_token<0, INTER, META, kBlockQ, NT>(a, meta, t, kRowQ, (w - t * a.parts_q) * kBlockQ, tab[wave]);
}

constexpr int kBlockWaves = 8;

template <bool INTER, int META, bool NT>
__global__ __launch_bounds__(64 * kBlockWaves) void block_append_kernel(const RopeAppend a) {
    block_append_body<INTER, META, NT>(a, a.meta);
}
template <bool INTER, int N>
__global__ __launch_bounds__(64 * kBlockWaves) void block_append_inline_kernel(const RopeInline<N> x) {
    const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    block_append_body<INTER, kMetaList, false>(x.a, reinterpret_cast<const int32_t*>(args + offsetof(RopeInline<N>, meta)));
}

int groups(int heads) { return (heads + kRows - 1) / kRows; }

// A large call's waves take up to kManyU groups of four rows (the turns are worked
// out once a wave), a small one's one each (more waves, shorter ones). Same box, us,
// 8192 tokens of 32 + 8 heads at 2, 3, 4, 5, 6, 12 groups: 35.0, 34.6, 32.7, 32.9,
// 34.2, 38.7. One group and four: 128 tokens (1280 groups) 2.7 / 3.4, 800 (8000) 4.7 /
// 5.2, 1200 (12000) 6.9 / 6.3, 3200 14.8 / 12.2; into fp16 pages 256 tokens (12 groups
// each) 3.6 / 3.8, 512 4.6 / 4.3, 1024 7.8 / 6.1. So calls without a cache cross near
// 8192 groups, appends of these heads between 256 and 512 tokens, 4000 groups or so:
// one border for both costs 512 of them 0.3 us.
constexpr int  kManyU      = 4;
constexpr long kManyGroups = 8192;

// Whether a call's loads bypass the caches: from some 100 MB of rows on, which the
// projection before it cannot have left in the memory-side cache (256 MB, the
// outputs beside them), and where a load takes whole 128-byte lines, which partial
// half-split rotations do not. us with cached and with non-temporal loads: 3200
// tokens of 32 + 8 heads (33 MB) 12.0 / 14.0, 6400 (66) 21.8 / 24.7, 8600 (88) 31.5 /
// 31.2, 9830 (101, the border) 34.1 / 35.5, 11000 (113) 39.1 / 38.8, 12800 (131) 45.6 /
// 44.8; with 8 more heads of values into FP8 pages 7200 (88) 29.0 / 30.4, 8192 (101)
// 34.0 / 34.3, 9400 (116) 39.8 / 38.7, 10700 (131) 44.7 / 43.8; into block-scaled ones
// 6200 (76) 25.7 / 29.3, 8192 38.2 / 37.0, 10700 48.6 / 45.9, 32768 (403) 145 / 137; with
// 96 of 128 dims turned 8192 of 32 + 8 29.0 / 36.4.
constexpr long kStreamBytes = 96l << 20;

// Parts of a token at u groups a wave, and the grid.
dim3 rows_grid(RopeAppend& a, bool cache, int u) {
    a.parts_q = (groups(a.q.heads) + u - 1) / u;
    a.parts_k = (groups(a.k.heads) + u - 1) / u;
    a.parts   = a.parts_q + (cache ? 2 : 1) * a.parts_k;
    a.by_page  = page_div(std::max(a.page_size, 1));
    a.by_parts = page_div(a.parts);
    a.ent_rate = static_cast<float>(a.n_ent) / static_cast<float>(a.n_tok);
    const long waves = static_cast<long>(a.n_tok) * a.parts;
    return dim3(static_cast<unsigned>((waves + kRowWaves - 1) / kRowWaves));
}
bool many(const RopeAppend& a, bool cache) {
    return static_cast<long>(a.n_tok) * (groups(a.q.heads) + (cache ? 2 : 1) * groups(a.k.heads)) >= kManyGroups;
}

bool streams(const RopeAppend& a, bool cache) {
    const bool lines = a.rope.interleaved || a.rope.pairs == 0 || a.rope.pairs == kPairs;
    const long rows  = static_cast<long>(a.n_tok) * (a.q.heads + (cache ? 2 : 1) * a.k.heads);
    return lines && rows * kRowBytes<2> >= kStreamBytes;
}

template <int CACHE, bool INTER, int META>
void launch_rows_i(RopeAppend a, hipStream_t s) {
    const dim3 block(64 * kRowWaves);
    if (many(a, CACHE != 0)) {
        const dim3 grid = rows_grid(a, CACHE != 0, kManyU);
        if (streams(a, CACHE != 0))
            hipLaunchKernelGGL((head_rows_kernel<CACHE, INTER, META, kManyU, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((head_rows_kernel<CACHE, INTER, META, kManyU, false>), grid, block, 0, s, a);
    } else {
        const dim3 grid = rows_grid(a, CACHE != 0, 1);
        hipLaunchKernelGGL((head_rows_kernel<CACHE, INTER, META, 1, false>), grid, block, 0, s, a);
    }
}
template <int CACHE, int META>
void launch_rows(const RopeAppend& a, hipStream_t s) {
    if (a.rope.interleaved) launch_rows_i<CACHE, true, META>(a, s);
    else launch_rows_i<CACHE, false, META>(a, s);
}
template <int CACHE, bool INTER, int N>
void launch_rows_inline_i(const RopeAppend& a, const int32_t* meta, size_t n, hipStream_t s) {
    RopeInline<N> x;
    x.a = a;
    std::copy(meta, meta + n, x.meta);
    const dim3 block(64 * kRowWaves);
    if (many(a, true)) {
        const dim3 grid = rows_grid(x.a, true, kManyU);
        hipLaunchKernelGGL((head_rows_inline_kernel<CACHE, INTER, kManyU, N>), grid, block, 0, s, x);
    } else {
        const dim3 grid = rows_grid(x.a, true, 1);
        hipLaunchKernelGGL((head_rows_inline_kernel<CACHE, INTER, 1, N>), grid, block, 0, s, x);
    }
}
template <int CACHE, int N>
void launch_rows_inline(const RopeAppend& a, const int32_t* meta, size_t n, hipStream_t s) {
    if (a.rope.interleaved) launch_rows_inline_i<CACHE, true, N>(a, meta, n, s);
    else launch_rows_inline_i<CACHE, false, N>(a, meta, n, s);
}

// Waves of a block and blocks of a block_append_kernel launch; sets a.units.
dim3 block_grid(RopeAppend& a, int& waves) {
    waves = std::min(a.k.heads, kBlockWaves);
    const int b   = block_tokens(a.page_size);
    a.block_shift = b == 16 ? 4 : 3;
    a.by_token    = a.n_tok <= a.n_tok / b + 2 * a.n_ent;
    a.units       = a.by_token ? a.n_tok : a.n_tok / b + 2 * a.n_ent;
    a.head_groups = (a.k.heads + waves - 1) / waves;
    a.parts_q     = (groups(a.q.heads) + kBlockQ - 1) / kBlockQ;
    a.by_page     = page_div(a.page_size);
    a.by_parts    = page_div(std::max(a.parts_q, 1));
    a.ent_rate    = static_cast<float>(a.n_ent) / static_cast<float>(a.units);
    const long q = static_cast<long>(a.n_tok) * a.parts_q;
    return dim3(static_cast<unsigned>(2l * a.units * a.head_groups + (q + waves - 1) / waves));
}
template <int META>
void launch_block(RopeAppend a, hipStream_t s) {
    int waves = 0;
    const dim3 grid = block_grid(a, waves), block(64 * waves);
    const bool nt = streams(a, true);
    if (a.rope.interleaved) {
        if (nt) hipLaunchKernelGGL((block_append_kernel<true, META, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_append_kernel<true, META, false>), grid, block, 0, s, a);
    } else {
        if (nt) hipLaunchKernelGGL((block_append_kernel<false, META, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_append_kernel<false, META, false>), grid, block, 0, s, a);
    }
}
template <int N>
void launch_block_inline(const RopeAppend& a, const int32_t* meta, size_t n, hipStream_t s) {
    RopeInline<N> x;
    x.a = a;
    std::copy(meta, meta + n, x.meta);
    int waves = 0;
    const dim3 grid = block_grid(x.a, waves), block(64 * waves);
    if (a.rope.interleaved) hipLaunchKernelGGL((block_append_inline_kernel<true, N>), grid, block, 0, s, x);
    else hipLaunchKernelGGL((block_append_inline_kernel<false, N>), grid, block, 0, s, x);
}

}  // namespace

hipError_t launch_norm_rope(const RopeAppend& a, hipStream_t s) {
    if (a.n_tok <= 0 || a.q.heads + a.k.heads == 0) return hipSuccess;
    launch_rows<0, 0>(a, s);
    return hipGetLastError();
}

hipError_t launch_append_rope(int dtype, const RopeAppend& a, const int32_t* meta, size_t n_meta, hipStream_t s) {
    check_kv_dtype(dtype);
    if (a.n_tok <= 0) return hipSuccess;
    const bool list  = a.meta != nullptr;   // a cache's append, its meta too long for the arguments
    const bool small = meta && n_meta <= 256;
    if (dtype == PA_KV_FP8_E4M3_BLOCK) {
        if (small) launch_block_inline<256>(a, meta, n_meta, s);
        else if (meta) launch_block_inline<kRopeInlineInts>(a, meta, n_meta, s);
        else if (list) launch_block<kMetaList>(a, s);
        else launch_block<kMetaTable>(a, s);
    } else if (dtype == PA_KV_FP16) {
        if (small) launch_rows_inline<1, 256>(a, meta, n_meta, s);
        else if (meta) launch_rows_inline<1, kRopeInlineInts>(a, meta, n_meta, s);
        else if (list) launch_rows<1, kMetaList>(a, s);
        else launch_rows<1, kMetaTable>(a, s);
    } else {
        if (small) launch_rows_inline<2, 256>(a, meta, n_meta, s);
        else if (meta) launch_rows_inline<2, kRopeInlineInts>(a, meta, n_meta, s);
        else if (list) launch_rows<2, kMetaList>(a, s);
        else launch_rows<2, kMetaTable>(a, s);
    }
    return hipGetLastError();
}

}  // namespace pa
