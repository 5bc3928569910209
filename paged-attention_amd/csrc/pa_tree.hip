// gfx950 attention of several new tokens per sequence over a paged cache: drafted
// trees, chains, pieces of prompts.

#include "pa_device.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

namespace pa {
namespace {

typedef float    f32x16 __attribute__((ext_vector_type(16)));
typedef float    f32x2  __attribute__((ext_vector_type(2)));
typedef short    s16x4  __attribute__((ext_vector_type(4)));

constexpr int kSub     = 32;              // places of one MFMA step
constexpr int kWavesT  = 4;
constexpr int kThreads = 64 * kWavesT;
constexpr int kOutLd   = kHeadDim + 4;    // floats of a row in the joining of waves

// A probability is kept as 2^(score - reference + kShift) in fp16, where the reference
// follows the row's maximum with a lag of at most kLag: 2^14 at most, and normal down
// to 2^-20 of the maximum (fp16 is subnormal below 2^-14).
constexpr float kShift = 6.0f;
constexpr float kLag   = 8.0f;

struct Entry {
    int t0, n, start, row;
};

// Entry e as the launch may use it: no tokens where it is out of range.
__device__ __forceinline__ Entry entry_at(const CachedTokens& c, int e) {
    Entry x;
    x.t0    = load_uniform(c.tok_begin, e);
    x.n     = min(load_uniform(c.tok_begin, e + 1), c.n_tok) - x.t0;
    x.start = load_uniform(c.start, e);
    x.row   = c.slot_ids ? load_uniform(c.slot_ids, e) : e;
    const bool ok = x.t0 >= 0 && x.n > 0 && x.start >= 0 && x.row >= 0 && x.row < c.table_rows &&
                    static_cast<long>(x.start) + x.n <= min(static_cast<long>(c.table_stride) * c.page_size, static_cast<long>(INT_MAX - kSub * kWavesT));
    if (!ok) x.n = 0;
    return x;
}
// The same per lane.
__device__ __forceinline__ Entry entry_of_lane(const CachedTokens& c, int e) {
    Entry x;
    x.t0    = c.tok_begin[e];
    x.n     = min(c.tok_begin[e + 1], c.n_tok) - x.t0;
    x.start = c.start[e];
    x.row   = c.slot_ids ? c.slot_ids[e] : e;
    const bool ok = x.t0 >= 0 && x.n > 0 && x.start >= 0 && x.row >= 0 && x.row < c.table_rows &&
                    static_cast<long>(x.start) + x.n <= min(static_cast<long>(c.table_stride) * c.page_size, static_cast<long>(INT_MAX - kSub * kWavesT));
    if (!ok) x.n = 0;
    return x;
}

// Units of work of an entry and one kv head: tiles of rows, times the steps over the
// places where items are split.
__device__ __forceinline__ long entry_cost(const TreeAttention& a, const Entry& x, int step) {
    if (x.n == 0) return 0;
    const long tiles = (x.n + a.tile_tokens - 1) / a.tile_tokens;
    return tiles * a.c.hkv * (a.split ? (x.start + x.n + step - 1) / step : 1);
}

struct Schedule {
    long pre[kThreads + 1];   // units before each entry of the chunk
    long wave_sum[kWavesT];
    int  hit;
};

// The units of entries c0 .. c0 + 255 as a running sum in s.pre.
__device__ long scan_chunk(const TreeAttention& a, Schedule& s, int c0, int step) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.c.n_ent == 1) {
        const long one = entry_cost(a, entry_at(a.c, 0), step);
        __syncthreads();
        s.pre[tid + 1] = one;
        if (tid == 0) s.pre[0] = 0;
        __syncthreads();
        return one;
    }
    long x = c0 + tid < a.c.n_ent ? entry_cost(a, entry_of_lane(a.c, c0 + tid), step) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s.wave_sum[wave] = x;
    __syncthreads();
    long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWavesT; ++w) {
        if (w < wave) before += s.wave_sum[w];
        total += s.wave_sum[w];
    }
    s.pre[tid + 1] = before + x;
    if (tid == 0) s.pre[0] = 0;
    __syncthreads();
    return total;
}

// LDS chunk (16 bytes) of a row that holds its chunk ch: rows that a fragment read takes
// together lie in different banks (K: 16 rows, one chunk; V: 4 rows, 4 chunks).
__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

__device__ __forceinline__ void block_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ float max_halves(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];   // (a bit_cast of a vector's element takes its first)
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float add_halves(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

__device__ __forceinline__ uint32_t ones(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// Which of the 32 places from j0 on (counted from the entry's first token) token i of an
// entry sees: every earlier one, and of the entry's n those that its tree row names.
__device__ __forceinline__ uint32_t visible(const TreeAttention& a, const Entry& x, int i, int j0) {
    if (i >= x.n) return 0;
    if (!a.tree) return ones(i - j0 + 1);
    const uint64_t* row = a.tree + static_cast<size_t>(x.t0 + i) * a.words;
    uint32_t bits;
    if (j0 < 0) {
        bits = ones(-j0);
        if (j0 > -32) bits |= static_cast<uint32_t>(row[0] << -j0);
    } else {
        const int w = j0 >> 6, sh = j0 & 63;
        uint64_t v = w < a.words ? row[w] >> sh : 0;
        if (sh > 32 && w + 1 < a.words) v |= row[w + 1] << (64 - sh);
        bits = static_cast<uint32_t>(v);
    }
    return bits & ones(x.n - j0);
}

// EB: bytes of a cached value; BS: block scales. 32 RQ rows a wave, WQ waves of rows,
// WK waves along the places.
template <int EB, bool BS, int RQ, int WQ, int WK>
struct TreeKernel {
    static constexpr int kRowsM = 32 * RQ * WQ;
    static constexpr int kStep  = kSub * WK;
    static constexpr int NJ     = 8 / WQ;              // 8-dim chunks of K (and of V) per thread and step
    static constexpr int kBufs  = WQ > 1 ? 2 : 1;
    static constexpr int kTile  = kSub * 256;          // bytes of 32 rows in fp16
    static constexpr int kStage = WK * kBufs * (2 * kTile + (BS ? 128 : 0));
    static constexpr int kJoin  = kWavesT * 32 * kOutLd * 4 + kWavesT * 32 * 8;
    static constexpr int kLds   = kStage > kJoin ? kStage : kJoin;

    typedef uint32_t Raw __attribute__((ext_vector_type(EB == 2 ? 4 : 2)));

    static __device__ __forceinline__ void run(const TreeAttention& a, unsigned char* lds, Schedule& sch) {
        const long step = kStep;
        // The block's share of the units, consecutive ones on one XCD (blocks go round the 8 XCDs).
        const int nb = gridDim.x;
        const int lb = nb % 8 == 0 ? (blockIdx.x % 8) * (nb / 8) + blockIdx.x / 8 : blockIdx.x;
        long total = 0, chunk = 0;
        for (int c0 = 0; c0 < a.c.n_ent; c0 += kThreads) total += chunk = scan_chunk(a, sch, c0, kStep);
        const long per = a.split ? max((total + nb - 1) / nb, 1l) : 1;
        long w = lb * per;
        const long w_end = min(w + per, total);
        if (w >= w_end) return;
        int  c0 = 0;
        long before = 0;
        if (a.c.n_ent > kThreads) chunk = scan_chunk(a, sch, 0, kStep);
        const long w_first = w;
        while (w < w_end) {
            while (w >= before + chunk) {
                before += chunk;
                c0 += kThreads;
                chunk = scan_chunk(a, sch, c0, kStep);
            }
            if (sch.pre[threadIdx.x] <= w - before && w - before < sch.pre[threadIdx.x + 1]) sch.hit = threadIdx.x;
            __syncthreads();
            const int  hit = a.c.n_ent == 1 ? 0 : __builtin_amdgcn_readfirstlane(sch.hit);
            const long at  = before + sch.pre[hit];
            __syncthreads();
            const Entry x = entry_at(a.c, c0 + hit);
            const int tiles = (x.n + a.tile_tokens - 1) / a.tile_tokens;
            const int steps = static_cast<int>((x.start + x.n + step - 1) / step);
            const int units = a.split ? steps : 1;
            const long local = w - at;
            const long item  = local / units;
            const int  u0    = static_cast<int>(local - item * units);
            const int  u1    = static_cast<int>(min(static_cast<long>(units), u0 + (w_end - w)));
            const int  h     = static_cast<int>(item / tiles);
            const int  rt    = tiles - 1 - static_cast<int>(item - static_cast<long>(h) * tiles);
            const bool whole = u0 == 0 && u1 == units;
            if (a.split && u0 == 0) {
                // For the merge: where the item's parts lie.
                const long b0 = w / per, b1 = (at + (item + 1) * units - 1) / per;
                const int  n  = min(a.tile_tokens, x.n - rt * a.tile_tokens);
                for (int i = threadIdx.x; i < n; i += kThreads) {
                    int32_t* d = a.desc + 2 * (static_cast<size_t>(x.t0 + rt * a.tile_tokens + i) * a.c.hkv + h);
                    d[0] = static_cast<int>(2 * b0 + (w == w_first ? 0 : 1));
                    d[1] = static_cast<int>(b1 - b0 + 1);
                }
            }
            const int slot = whole ? -1 : 2 * lb + (w == w_first ? 0 : 1);
            item_part(a, lds, x, h, rt, a.split ? u0 : 0, a.split ? u1 : steps, slot);
            w += u1 - u0;
        }
    }

    static __device__ __forceinline__ void item_part(const TreeAttention& a, unsigned char* lds, const Entry& x, int h,
                                                     int rt, int k0, int k1, int slot) {
        const CachedTokens& c = a.c;
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave % WQ, wk = wave / WQ;
        const int ql = lane & 31, hl = lane >> 5;
        const int G = a.group, P = c.page_size;
        const int tok0 = rt * a.tile_tokens;   // first token of the tile, within the entry
        const int tile_n = min(a.tile_tokens, x.n - tok0);
        const int end = x.start + (a.tree ? x.n : tok0 + tile_n);   // places from here on are not seen
        k1 = min(k1, (end + kStep - 1) / kStep);

        // Query fragments, and each lane's token.
        f16x8 q[RQ][8];
        int   tok[RQ];
#pragma unroll
        for (int r = 0; r < RQ; ++r) {
            const int row = 32 * (RQ * wq + r) + ql;
            const int i = a.by_group.page(row), g = row - i * G;
            const bool ok = i < tile_n;
            tok[r] = ok ? tok0 + i : INT_MAX;
            const uint16_t* p = a.q + (x.t0 + tok0 + (ok ? i : 0)) * a.q_stride + (h * G + (ok ? g : 0)) * kHeadDim + 8 * hl;
#pragma unroll
            for (int s = 0; s < 8; ++s) q[r][s] = __builtin_bit_cast(f16x8, *reinterpret_cast<const u32x4*>(p + 16 * s));
        }
        // First token of the wave's rows: what it sees all of them see, in a chain.
        const int first_tok = tok0 + a.by_group.page(32 * RQ * wq);

        f32x16 o[RQ][4];
        float  m[RQ], l[RQ];
#pragma unroll
        for (int r = 0; r < RQ; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[r][d][i] = 0.f;
        }

        // Staging: this thread's rows row0 + 4 WQ j of a step's 32, chunk ch of each.
        const int gt = 64 * wq + lane, row0 = gt >> 4, ch = gt & 15;
        const int32_t* table = c.table + static_cast<size_t>(x.row) * c.table_stride;
        const size_t page_bytes = static_cast<size_t>(c.hkv) * P * kRowBytes<EB>;
        const size_t head_off   = static_cast<size_t>(h) * P * kRowBytes<EB> + ch * 8 * EB;
        const int    bsh = BS ? (P % 16 == 0 ? 4 : 3) : 0, nblk = BS ? P >> bsh : 0;
        int      pg[NJ];
        Raw      kr[NJ], vr[NJ];
        uint32_t sc[NJ];
        uint32_t live = 0;   // rows of kr / vr that hold a place
        auto lookup = [&](int k) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int t = k * kStep + kSub * wk + row0 + 4 * WQ * j;
                pg[j] = t < end ? table[c.by_page.page(t)] : -1;
            }
        };
        auto issue = [&](int k) {
            live = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int t = k * kStep + kSub * wk + row0 + 4 * WQ * j;
                const bool ok = pg[j] >= 0 && pg[j] < c.num_pages;
                live |= ok ? 1u << j : 0u;
                const int page = ok ? pg[j] : 0, s = ok ? t - c.by_page.page(t) * P : 0;
                const size_t off = page * page_bytes + head_off + static_cast<size_t>(s) * kRowBytes<EB>;
                kr[j] = *reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(c.k_cache) + off);
                vr[j] = *reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(c.v_cache) + off);
                if constexpr (BS)
                    sc[j] = *reinterpret_cast<const uint16_t*>(c.scales + 2 * ((static_cast<size_t>(page) * c.hkv + h) * nblk + (s >> bsh)));
            }
        };
        auto widen = [](Raw x, float scale) {
            if constexpr (EB == 2) return x;
            else return u32x4{fp8x2_to_f16x2<false>(x[0], scale), fp8x2_to_f16x2<true>(x[0], scale),
                              fp8x2_to_f16x2<false>(x[1], scale), fp8x2_to_f16x2<true>(x[1], scale)};
        };
        auto stage_at = [&](int buf) { return lds + (wk * kBufs + buf) * (2 * kTile + (BS ? 128 : 0)); };
        auto store = [&](int buf) {
            unsigned char* k = stage_at(buf);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int row = row0 + 4 * WQ * j;
                const bool ok = live >> j & 1;
                const float vs = BS ? __builtin_bit_cast(float, (sc[j] >> 8) << 23) : 1.0f;
                u32x4 kx = widen(kr[j], 1.0f), vx = widen(vr[j], vs);
                if (!ok) kx = vx = u32x4{0, 0, 0, 0};
                const int at = row * 256 + ((ch ^ swizzle(row)) << 4);
                *reinterpret_cast<u32x4*>(k + at) = kx;
                *reinterpret_cast<u32x4*>(k + kTile + at) = vx;
                if constexpr (BS)
                    if (ch == 0)
                        *reinterpret_cast<float*>(k + 2 * kTile + 4 * row) = __builtin_bit_cast(float, (sc[j] & 0xff) << 23);
            }
        };

        // Where this lane's fragments lie in the stage.
        const int ka = ql * 256 + ((hl ^ swizzle(ql)) << 4);
        const int vi = lane & 15, vg = (lane >> 4) & 1;
        const int va = (4 * hl + (vi >> 2)) * 256 + ((((vi >> 2) << 2) | ((2 * vg + ((vi >> 1) & 1)) ^ hl)) << 4) + 8 * (vi & 1);

        auto compute = [&](int k, int buf) {
            const int base = k * kStep + kSub * wk;
            if (base >= end) return;
            const unsigned char* ks = stage_at(buf);
            const unsigned char* vs = ks + kTile;
            f32x16 s[RQ];
#pragma unroll
            for (int r = 0; r < RQ; ++r)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[r][i] = 0.f;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const f16x8 kf = *reinterpret_cast<const f16x8*>(ks + (ka ^ (t << 5)));
#pragma unroll
                for (int r = 0; r < RQ; ++r) s[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[r][t], s[r], 0, 0, 0);
            }
            float cs[4];   // base-2 scores of a raw product, per eight places
#pragma unroll
            for (int i = 0; i < 4; ++i)
                cs[i] = BS ? a.score_scale * *reinterpret_cast<const float*>(ks + 2 * kTile + 32 * i) : a.score_scale;
            const bool masked = base + kSub > x.start + (a.tree ? 0 : first_tok + 1);
            uint32_t seen[RQ];
            f16x8    p[RQ][2];
#pragma unroll
            for (int r = 0; r < RQ; ++r) {
                seen[r] = ~0u;
                if (masked) {
                    seen[r] = visible(a, x, tok[r], base - x.start);
                    const uint32_t mine = seen[r] >> (4 * hl);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[r][i] = mine >> (8 * (i / 4) + i % 4) & 1 ? s[r][i] * cs[i / 4] : -INFINITY;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[r][i] *= cs[i / 4];
                }
                float top = s[r][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, s[r][i]);
                top = max_halves(top);
                if (__builtin_amdgcn_ballot_w64(top > m[r] + kLag) != 0) {
                    const float now = fmaxf(m[r], top), ref = now == -INFINITY ? 0.f : now;
                    const float f = exp2_fast(m[r] - ref);
                    l[r] *= f;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[r][d][i] *= f;
                    m[r] = now;
                }
                const float ref = (m[r] == -INFINITY ? 0.f : m[r]) - kShift;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = exp2_fast(s[r][i] - ref);
                    l[r] += e;
                    p[r][i / 8][i % 8] = static_cast<_Float16>(e);
                }
            }
            auto v_part = [&](int d, int u, int w) {
                const int at = (va ^ (d << 6) ^ (w << 5)) + (16 * u + 8 * w) * 256;
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vs + at));
            };
            auto v_frag = [&](int d, int u) {
                const s16x4 lo = v_part(d, u, 0), hi = v_part(d, u, 1);
                return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            if (!masked) {
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const f16x8 v = v_frag(d, u);
#pragma unroll
                        for (int r = 0; r < RQ; ++r)
                            o[r][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[r][u], o[r][d], 0, 0, 0);
                    }
                return;
            }
            // A place that a row does not see must not reach it, whatever its value: 0 * infinity
            // is NaN. Values that are not finite are taken as zeros, and then added as such to the
            // rows that see them: how many of each sign a row sees comes from two more products.
            uint32_t odd = 0;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    f16x8 v = v_frag(d, u);
                    u32x4 b = __builtin_bit_cast(u32x4, v);
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 8; ++e) bad |= (b[e / 2] >> (16 * (e & 1)) & 0x7c00u) == 0x7c00u;
                    if (__builtin_amdgcn_ballot_w64(bad) != 0) {
                        odd |= 1u << d;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((b[e / 2] >> (16 * (e & 1)) & 0x7c00u) == 0x7c00u) v[e] = static_cast<_Float16>(0.f);
                    }
#pragma unroll
                    for (int r = 0; r < RQ; ++r)
                        o[r][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[r][u], o[r][d], 0, 0, 0);
                }
            if (odd == 0) return;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                if (!(odd >> d & 1)) continue;
#pragma unroll
                for (int r = 0; r < RQ; ++r) {
                    const uint32_t mine = seen[r] >> (4 * hl);
#pragma unroll
                    for (int sign = 0; sign < 2; ++sign) {
                        f32x16 n = {};
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const u32x4 b = __builtin_bit_cast(u32x4, v_frag(d, u));
                            f16x8 is, sees;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const uint32_t y = b[e / 2] >> (16 * (e & 1)) & 0xffffu;
                                const bool hit = (y & 0x7fffu) > 0x7c00u || y == (sign ? 0xfc00u : 0x7c00u);
                                const int  i = 8 * u + e;
                                is[e]   = static_cast<_Float16>(hit ? 1.f : 0.f);
                                sees[e] = static_cast<_Float16>(mine >> (8 * (i / 4) + i % 4) & 1 ? 1.f : 0.f);
                            }
                            n = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, sees, n, 0, 0, 0);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (n[i] > 0.f) o[r][d][i] += sign ? -INFINITY : INFINITY;
                    }
                }
            }
        };

        if (k0 < k1) {
            lookup(k0);
            issue(k0);
            if (k0 + 1 < k1) lookup(k0 + 1);
        }
        for (int k = k0; k < k1; ++k) {
            const int buf = kBufs == 2 ? (k - k0) & 1 : 0;
            store(buf);
            if (k + 1 < k1) {
                issue(k + 1);
                if (k + 2 < k1) lookup(k + 2);
            }
            if constexpr (WQ > 1) block_sync();
            else wave_lds_sync();
            compute(k, buf);
            if constexpr (WQ == 1) wave_lds_sync();
        }

        // The waves along the places joined, through LDS, 32 rows of each wave at a time.
        float* const ol = reinterpret_cast<float*>(lds);
        float* const ml = ol + kWavesT * 32 * kOutLd;
#pragma unroll
        for (int r = 0; r < RQ; ++r) {
            const float sum = add_halves(l[r]);
            __syncthreads();
            float* mine = ol + (32 * wave + ql) * kOutLd;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(mine + 32 * d + 8 * i + 4 * hl) =
                        f32x4{o[r][d][4 * i], o[r][d][4 * i + 1], o[r][d][4 * i + 2], o[r][d][4 * i + 3]};
            if (hl == 0) *reinterpret_cast<f32x2*>(ml + 2 * (32 * wave + ql)) = f32x2{m[r], sum};
            __syncthreads();
            constexpr int TR = kThreads / (32 * WQ);   // threads of a row
            const int jr = tid / TR, part = tid % TR;  // row among 32 WQ; a quarter-dims of it
            const int w0 = jr / 32, row = 32 * (RQ * w0 + r) + jr % 32;
            float top = -INFINITY, den = 0.f;
            float f[WK];
#pragma unroll
            for (int g = 0; g < WK; ++g) top = fmaxf(top, ml[2 * (32 * (g * WQ + w0) + jr % 32)]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int g = 0; g < WK; ++g) {
                const float* e = ml + 2 * (32 * (g * WQ + w0) + jr % 32);
                f[g] = exp2_fast(e[0] - ref);
                den += f[g] * e[1];
            }
            const int i = a.by_group.page(row), g0 = row - i * G;
            if (i < tile_n) {
                const float scale = slot >= 0 ? 1.f : den == 0.f ? 0.f : c.v_scale / den;
                uint16_t* out = a.out + (x.t0 + tok0 + i) * a.out_stride + (h * G + g0) * kHeadDim;
                float* po = slot >= 0 ? a.part_out + (static_cast<size_t>(slot) * kRowsM + row) * kHeadDim : nullptr;
#pragma unroll
                for (int d = 4 * part; d < kHeadDim; d += 4 * TR) {
                    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int g = 0; g < WK; ++g) {
                        const f32x4 z = *reinterpret_cast<const f32x4*>(ol + (32 * (g * WQ + w0) + jr % 32) * kOutLd + d);
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = fmaf(z[e], f[g], y[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] *= scale;
                    if (slot >= 0) {
                        *reinterpret_cast<f32x4*>(po + d) = y;
                    } else {
                        const f16x2 lo = {static_cast<_Float16>(y[0]), static_cast<_Float16>(y[1])};
                        const f16x2 hi = {static_cast<_Float16>(y[2]), static_cast<_Float16>(y[3])};
                        *reinterpret_cast<u32x2*>(out + d) =
                            u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
                    }
                }
                if (slot >= 0 && part == 0)
                    *reinterpret_cast<f32x2*>(a.part_ml + 2 * (static_cast<size_t>(slot) * kRowsM + row)) = f32x2{ref == 0.f && top == -INFINITY ? -INFINITY : ref, den};
            }
        }
        __syncthreads();   // the stage is free again
    }
};

template <int EB, bool BS, int RQ, int WQ, int WK>
__global__ __launch_bounds__(kThreads) void tree_attention_kernel(const TreeAttention a) {
    using T = TreeKernel<EB, BS, RQ, WQ, WK>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[T::kLds];
    __shared__ Schedule sch;
    T::run(a, lds, sch);
}

// Rows whose item was split: their parts joined. A wave a row.
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(const TreeAttention a) {
    const CachedTokens& c = a.c;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long id = static_cast<long>(blockIdx.x) * kWavesT + wave;
    const int hq = c.hkv * a.group;
    const int t = static_cast<int>(id / hq), head = static_cast<int>(id - static_cast<long>(t) * hq);
    if (t >= c.n_tok) return;
    // The token's entry: the last that begins at or before it.
    int lo = 0;
    for (int span = c.n_ent; span > 1;) {
        const int step = (span + 63) / 64, i = lo + step * lane;
        const bool le = i < lo + span && c.tok_begin[i] <= t;
        const int at = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(le)) - 1, 0);
        const int end = lo + span;
        lo += step * at;
        span = min(step, end - lo);
    }
    const Entry x = entry_at(c, lo);
    if (t < x.t0 || t >= x.t0 + x.n) return;
    const int h = head / a.group, g = head - h * a.group;
    const int32_t* d = a.desc + 2 * (static_cast<size_t>(t) * c.hkv + h);
    const int slot0 = d[0], n = d[1];
    if (n <= 1) return;
    const int row = (t - x.t0) % a.tile_tokens * a.group + g;
    f32x2 acc = {0.f, 0.f};
    float m = -INFINITY, den = 0.f;
    for (int k = 0; k < n; ++k) {
        const int    slot = k == 0 ? slot0 : 2 * (slot0 / 2 + k);
        const size_t at = static_cast<size_t>(slot) * a.rows + row;
        const f32x2  e = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * at);
        const f32x2  y = *reinterpret_cast<const f32x2*>(a.part_out + at * kHeadDim + 2 * lane);
        const float now = fmaxf(m, e[0]), ref = now == -INFINITY ? 0.f : now;
        const float f0 = exp2_fast(m - ref), f1 = exp2_fast(e[0] - ref);
        acc[0] = acc[0] * f0 + y[0] * f1;
        acc[1] = acc[1] * f0 + y[1] * f1;
        den = den * f0 + e[1] * f1;
        m = now;
    }
    const float scale = den == 0.f ? 0.f : c.v_scale / den;
    const f16x2 r = {static_cast<_Float16>(acc[0] * scale), static_cast<_Float16>(acc[1] * scale)};
    *reinterpret_cast<uint32_t*>(a.out + t * a.out_stride + head * kHeadDim + 2 * lane) = __builtin_bit_cast(uint32_t, r);
}

template <int EB, bool BS>
void launch_e(const TreeAttention& a, hipStream_t s) {
    const dim3 grid(a.grid), block(kThreads);
    switch (a.rows) {
        case 32: hipLaunchKernelGGL((tree_attention_kernel<EB, BS, 1, 1, 4>), grid, block, 0, s, a); break;
        case 64: hipLaunchKernelGGL((tree_attention_kernel<EB, BS, 2, 1, 4>), grid, block, 0, s, a); break;
        case 128: hipLaunchKernelGGL((tree_attention_kernel<EB, BS, 2, 2, 2>), grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL((tree_attention_kernel<EB, BS, 2, 4, 1>), grid, block, 0, s, a); break;
    }
}

int device_cus() {
    int dev = 0, n = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    hip_check(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev), "hipDeviceGetAttribute");
    return n;
}

}  // namespace

void tree_shape(int dtype, TreeAttention& a) {
    (void)dtype;
    const long per = (static_cast<long>(a.c.n_tok) * a.group + a.c.n_ent - 1) / std::max(a.c.n_ent, 1);   // rows of an entry
    a.rows        = per <= 32 && a.group <= 32 ? 32 : per <= 64 && a.group <= 64 ? 64 : per <= 128 ? 128 : 256;
    a.tile_tokens = a.rows / a.group;
    const long items = (static_cast<long>(a.c.n_tok) / a.tile_tokens + a.c.n_ent) * a.c.hkv;   // at most
    const int  cus = device_cus();
    a.split = items <= 16l * cus;
    a.grid  = a.split ? cus * (a.rows <= 32 ? 2 : 1) : static_cast<int>(items);
}

size_t tree_workspace(const TreeAttention& a) {
    if (!a.split) return 0;
    return static_cast<size_t>(2 * a.grid) * a.rows * (kHeadDim + 2) * sizeof(float) +
           static_cast<size_t>(a.c.n_tok) * a.c.hkv * 2 * sizeof(int32_t);
}

void tree_place(TreeAttention& a, void* workspace) {
    const size_t rows = static_cast<size_t>(2 * a.grid) * a.rows;
    a.part_out = static_cast<float*>(workspace);
    a.part_ml  = a.part_out + rows * kHeadDim;
    a.desc     = reinterpret_cast<int32_t*>(a.part_ml + 2 * rows);
}

hipError_t launch_tree_attention(int dtype, const TreeAttention& a, hipStream_t s) {
    check_kv_dtype(dtype);
    if (dtype == PA_KV_FP16) launch_e<2, false>(a, s);
    else if (dtype == PA_KV_FP8_E4M3) launch_e<1, false>(a, s);
    else launch_e<1, true>(a, s);
    if (a.split) {
        const long rows = static_cast<long>(a.c.n_tok) * a.c.hkv * a.group;
        hipLaunchKernelGGL(tree_merge_kernel, dim3(static_cast<unsigned>((rows + kWavesT - 1) / kWavesT)), dim3(kThreads), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace pa
