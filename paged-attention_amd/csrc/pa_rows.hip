// gfx950 kernels over rows of a paged cache: rows read back as numbers, and accepted
// drafted rows moved up in their sequences.
//
//   read_cache_kernel   places of several sequences out of the pages, side by side
//   keep_rows_kernel    accepted tokens' rows to the places behind one another
//   keep_blocks_kernel  the same in a block-scaled cache
//
// (No counterparts in the reference.)
//
// read_cache is bound by memory: a code in, its value (code times scale, in 32 bits, rounded once)
// out. 8 x 8192 places, block scales, into fp16: 74 us, 5.5 TB/s (the kernel over inputs that the last
// pass left in the caches: 59); 37 ragged sequences, FP8, 57 us (42). Of one kv head, 48 lanes of a
// wave have no row: 21 us for an eighth of the bytes. The keeping kernels move some rows of each sequence:
// a chain of loads (counts, numbers, pages, rows), and what its waves, one an entry and head, add. The kernels
// alone, 6 rows kept in 64 / 512 sequences: fp16 4.1 / 5.8 us, FP8 3.7 / 4.9, block scales 6.0 / 15; 16 rows: 5.1 / 9.4,
// 4.9 / 7.0, 6.2 / 20.

#include "pa_device.hpp"
#include "pa_fp8.hpp"

#include <algorithm>
#include <climits>
#include <cstdint>

namespace pa {
namespace {

constexpr int kWavesR = 4;
constexpr int kLanesR = 16;                // lanes of a row, 8 dims each
constexpr int kRowsR  = 64 / kLanesR;
constexpr int kHeadsR = 2;                // heads that a lane group has on their way

__device__ __forceinline__ float exp2_byte(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

// Entry that token t belongs to: the last that begins at or before it.
__device__ __forceinline__ int entry_of_token(const CachedTokens& c, int t) {
    int lo = 0;
    for (int span = c.n_ent; span > 1;) {
        const int step = (span + 63) / 64, i = lo + step * static_cast<int>(threadIdx.x & 63);
        const bool le = i < lo + span && c.tok_begin[i] <= t;
        const int at = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(le)) - 1, 0);
        const int end = lo + span;
        lo += step * at;
        span = min(step, end - lo);
    }
    return lo;
}

// Page of the place pos of a table row, -1 where there is none.
__device__ __forceinline__ int page_at(const CachedTokens& c, int row, int pos) {
    if (row < 0 || row >= c.table_rows || pos < 0) return -1;
    const int i = c.by_page.page(pos);
    if (i >= c.table_stride) return -1;
    const int page = c.table[static_cast<size_t>(row) * c.table_stride + i];
    return page >= 0 && page < c.num_pages ? page : -1;
}

// ---- reading back ----------------------------------------------------------

// (Streaming stores: outputs are the larger part of the traffic, and cached they push rows that are
// still to be read out of the caches. us with cached and with streaming stores: 8 x 8192 places,
// block scales, 84 / 61 on one input again and again, 84 / 74 on inputs in turn; 37 ragged sequences, FP8, 54 / 44 and
// 63 / 57.)
template <int OUT>
__device__ __forceinline__ void store_values(void* out, size_t at, const float (&y)[8]) {
    if constexpr (OUT == PA_VALUE_FP32) {
        float* p = static_cast<float*>(out) + at;
        __builtin_nontemporal_store(f32x4{y[0], y[1], y[2], y[3]}, reinterpret_cast<f32x4*>(p));
        __builtin_nontemporal_store(f32x4{y[4], y[5], y[6], y[7]}, reinterpret_cast<f32x4*>(p + 4));
    } else {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (OUT == PA_VALUE_FP16) {
                const f16x2 h = {static_cast<_Float16>(y[2 * e]), static_cast<_Float16>(y[2 * e + 1])};
                o[e] = __builtin_bit_cast(uint32_t, h);
            } else {
                typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                const bf16x2 h = {static_cast<__bf16>(y[2 * e]), static_cast<__bf16>(y[2 * e + 1])};
                o[e] = __builtin_bit_cast(uint32_t, h);
            }
        }
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + at));
    }
}

constexpr int kMaxReadBlocks = 1 << 22;   // in a row of the grid (a row holds fewer than 2^32 threads)

// A wave a token: its rows of every kv head, K's then V's.
template <int EB, bool BS, int OUT>
__global__ __launch_bounds__(64 * kWavesR) void read_cache_kernel(const ReadCache a) {
    const CachedTokens& c = a.c;
    const int lane = threadIdx.x & 63, ch = lane % kLanesR, r = lane / kLanesR;
    const int P = c.page_size, sh = BS ? (P % 16 == 0 ? 4 : 3) : 0;
    const int t = (blockIdx.y * gridDim.x + blockIdx.x) * kWavesR + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= c.n_tok) return;
    const int e = __builtin_amdgcn_readfirstlane(entry_of_token(c, t));
    const int t0 = load_uniform(c.tok_begin, e), t1 = load_uniform(c.tok_begin, e + 1), st = load_uniform(c.start, e);
    if (t < t0 || t >= t1 || st < 0 || st > INT_MAX - (t - t0)) return;
    const int pos  = st + (t - t0);
    const int page = page_at(c, c.slot_ids ? load_uniform(c.slot_ids, e) : e, pos);
    if (page < 0) return;
    const int slot = pos - c.by_page.page(pos) * P;
    typedef uint32_t Raw __attribute__((ext_vector_type(EB == 2 ? 4 : 2)));
    for (int h0 = r; h0 < c.hkv; h0 += kHeadsR * kRowsR) {
        Raw      x[kHeadsR][2];
        uint32_t sc[kHeadsR];
#pragma unroll
        for (int i = 0; i < kHeadsR; ++i) {
            const int h = min(h0 + kRowsR * i, c.hkv - 1);
            const size_t off = kv_row_offset<EB>(page, h, slot, P, c.hkv) + ch * 8 * EB;
            if (a.k_out) x[i][0] = *reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(c.k_cache) + off);
            if (a.v_out) x[i][1] = *reinterpret_cast<const Raw*>(static_cast<const unsigned char*>(c.v_cache) + off);
            sc[i] = 0;
            if constexpr (BS)
                sc[i] = *reinterpret_cast<const uint16_t*>(c.scales + 2 * ((static_cast<size_t>(page) * c.hkv + h) * (P >> sh) + (slot >> sh)));
        }
#pragma unroll
        for (int i = 0; i < kHeadsR; ++i) {
            const int h = h0 + kRowsR * i;
            if (h >= c.hkv) break;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                void* out = v ? a.v_out : a.k_out;
                if (!out) continue;
                f16x8 y16;
                if constexpr (EB == 2) y16 = __builtin_bit_cast(f16x8, x[i][v]);
                else y16 = fp8x8_to_f16x8(x[i][v][0], x[i][v][1]);
                // (A code times its block's scale is exact; the scales' product might not be, or past fp32.)
                const float f = BS ? exp2_byte(v ? sc[i] >> 8 : sc[i] & 0xff) : 1.f, g = v ? c.v_scale : c.k_scale;
                float y[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) y[d] = EB == 2 ? static_cast<float>(y16[d]) : static_cast<float>(y16[d]) * f * g;
                store_values<OUT>(out, t * (v ? a.v_stride : a.k_stride) + h * kHeadDim + ch * 8, y);
            }
        }
    }
}

// ---- keeping accepted rows -------------------------------------------------

// A wave an entry and kv head: rows of both pools in order, 16 at a time, read before they are
// stored; a row comes from its own place or a later one, so rows read later are not
// written by earlier stores.
template <int EB>
__global__ __launch_bounds__(64) void keep_rows_kernel(const KeepRows a) {
    typedef uint32_t Raw __attribute__((ext_vector_type(EB == 2 ? 4 : 2)));
    const CachedTokens& c = a.c;
    const int lane = threadIdx.x & 63, ch = lane % kLanesR, r = lane / kLanesR;
    const int e = blockIdx.x / c.hkv, h = blockIdx.x - e * c.hkv;
    unsigned char *kp = static_cast<unsigned char*>(c.k_cache), *vp = static_cast<unsigned char*>(c.v_cache);
    const int32_t* kept = a.kept + static_cast<size_t>(e) * a.width;
    int next[4];
    auto numbers = [&](int j0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + kRowsR * i + r;
            next[i] = j < a.width ? kept[j] : 0;
        }
    };
    numbers(0);
    const int n = min(load_uniform(a.counts, e), a.width), st = load_uniform(c.start, e);
    const int row = c.slot_ids ? load_uniform(c.slot_ids, e) : e;
    if (st < 0) return;
    for (int j0 = 0; j0 < n; j0 += 16) {
        Raw    x[4], y[4];
        size_t to[4];
        bool   ok[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + kRowsR * i + r, k = next[i];
            ok[i] = false;
            if (j >= n || k <= j || k > INT_MAX - st) continue;
            const int ps = page_at(c, row, st + k), pd = page_at(c, row, st + j);
            if (ps < 0 || pd < 0) continue;
            ok[i] = true;
            const size_t from = kv_row_offset<EB>(ps, h, st + k - c.by_page.page(st + k) * c.page_size, c.page_size, c.hkv) + ch * 8 * EB;
            x[i] = *reinterpret_cast<const Raw*>(kp + from);
            y[i] = *reinterpret_cast<const Raw*>(vp + from);
            to[i] = kv_row_offset<EB>(pd, h, st + j - c.by_page.page(st + j) * c.page_size, c.page_size, c.hkv) + ch * 8 * EB;
        }
        if (j0 + 16 < n) numbers(j0 + 16);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (ok[i]) {
                *reinterpret_cast<Raw*>(kp + to[i]) = x[i];
                *reinterpret_cast<Raw*>(vp + to[i]) = y[i];
            }
        asm volatile("" ::: "memory");
    }
}

__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    const int k = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(k, kBlockExpMin), kBlockExpMax);
}
__device__ __forceinline__ float wave_max64(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// Codes of y / 2^k for a row's 8 dims, the NaNs of `was` kept as they are.
__device__ __forceinline__ u32x2 recode(u32x2 was, float (&y)[8], int k) {
    const float inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inv;
    u32x2 now = e4m3_encode8(y, k == kBlockExpMax ? kBlockTop : 448.0f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t m = 0xffu << (8 * (i & 3));
        if ((was[i >> 2] >> (8 * (i & 3)) & 0x7fu) == 0x7fu) now[i >> 2] = (now[i >> 2] & ~m) | (was[i >> 2] & m);
    }
    return now;
}

constexpr int kWavesB = 2;

// Blocks of the places that the accepted rows come to, kWavesB at a time, a wave each: all are read
// before any is written. (A row comes from its own block or a later one, so what is read next has not
// been written.)
__global__ __launch_bounds__(64 * kWavesB) void keep_blocks_kernel(const KeepRows a) {
    const CachedTokens& c = a.c;
    const int lane = threadIdx.x & 63, ch = lane % kLanesR, r = lane / kLanesR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e = blockIdx.x / c.hkv, h = blockIdx.x - e * c.hkv, v = blockIdx.y;
    unsigned char* pool = static_cast<unsigned char*>(v ? c.v_cache : c.k_cache);
    const int n = min(load_uniform(a.counts, e), a.width), st = load_uniform(c.start, e);
    const int row = c.slot_ids ? load_uniform(c.slot_ids, e) : e;
    if (st < 0 || n <= 0) return;
    const int P = c.page_size, sh = P % 16 == 0 ? 4 : 3, B = 1 << sh, nb = P >> sh;
    const int last = (n - 1 > INT_MAX - st ? INT_MAX : st + n - 1) >> sh;
    const int32_t* kept = a.kept + static_cast<size_t>(e) * a.width;
    auto scale_at = [&](int page, int slot) {
        return c.scales + 2 * ((static_cast<size_t>(page) * c.hkv + h) * nb + (slot >> sh)) + v;
    };
    for (int b0 = st >> sh; b0 <= last; b0 += kWavesB) {
        // Lane group r holds the block's places r, r + 4, ...
        const int b = b0 + wave, at = b <= last ? b * B : -1, page = page_at(c, row, at);   // (none before place 0)
        const int slot0 = page < 0 ? 0 : at - c.by_page.page(at) * P;
        u32x2 was[4];
        int   from[4];     // 0: not in the path, 1: stays in its place, 2: moves in, 3: lies before the path
        float y[4][8], amax = 0.f;
        bool  moved = false;
        uint8_t* const sc = scale_at(max(page, 0), slot0);
        const int old = page < 0 ? 0 : *sc;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = kRowsR * i + r, j = max(at, 0) + s - st;
            from[i] = 0;
            was[i] = u32x2{0, 0};
            float f = 0.f;
            if (page >= 0 && s < B && j < n) {
                const int k = j < 0 ? j : kept[j];
                const int pos = st + k;
                const int ps = j >= 0 && (k < j || k > INT_MAX - st) ? -1 : k == j ? page : page_at(c, row, pos);
                if (ps >= 0) {
                    const int ss = pos - c.by_page.page(pos) * P;
                    was[i] = *reinterpret_cast<const u32x2*>(pool + kv_row_offset<1>(ps, h, ss, P, c.hkv) + ch * 8);
                    f = exp2_byte(*scale_at(ps, ss));
                    from[i] = j < 0 ? 3 : k == j ? 1 : 2;
                    moved |= from[i] == 2;
                }
            }
            const f16x8 g = fp8x8_to_f16x8(was[i][0], was[i][1]);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                y[i][d] = static_cast<float>(g[d]) * f;
                if (from[i] == 1 || from[i] == 2) amax = fmaxf(amax, fabsf(y[i][d]));
            }
        }
        __syncthreads();
        if (__builtin_amdgcn_ballot_w64(moved) == 0) continue;
        int k = __builtin_amdgcn_readfirstlane(block_exponent(wave_max64(amax)));
        if (at < st) k = max(k, old - 127);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (from[i] == 0 || (from[i] == 3 && k <= old - 127)) continue;
            *reinterpret_cast<u32x2*>(pool + kv_row_offset<1>(page, h, slot0 + kRowsR * i + r, P, c.hkv) + ch * 8) = recode(was[i], y[i], k);
        }
        if (lane == 0) *sc = static_cast<uint8_t>(k + 127);
    }
}

}  // namespace

template <int EB, bool BS>
void launch_read(int out_type, const ReadCache& a, hipStream_t s) {
    const int  n = (a.c.n_tok + kWavesR - 1) / kWavesR, x = std::min(n, kMaxReadBlocks);
    const dim3 grid(x, (n + x - 1) / x), block(64 * kWavesR);
    if (out_type == PA_VALUE_FP32) hipLaunchKernelGGL((read_cache_kernel<EB, BS, PA_VALUE_FP32>), grid, block, 0, s, a);
    else if (out_type == PA_VALUE_BF16) hipLaunchKernelGGL((read_cache_kernel<EB, BS, PA_VALUE_BF16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((read_cache_kernel<EB, BS, PA_VALUE_FP16>), grid, block, 0, s, a);
}

hipError_t launch_read_cache(int dtype, int out_type, const ReadCache& a, hipStream_t s) {
    check_kv_dtype(dtype);
    if (dtype == PA_KV_FP16) launch_read<2, false>(out_type, a, s);
    else if (dtype == PA_KV_FP8_E4M3) launch_read<1, false>(out_type, a, s);
    else launch_read<1, true>(out_type, a, s);
    return hipGetLastError();
}

int keep_threads(int dtype) { return dtype == PA_KV_FP8_E4M3_BLOCK ? 64 * kWavesB : 64; }

hipError_t launch_keep_rows(int dtype, const KeepRows& a, hipStream_t s) {
    check_kv_dtype(dtype);
    const dim3 grid(a.c.n_ent * a.c.hkv, 2), both(a.c.n_ent * a.c.hkv), block(keep_threads(dtype));
    if (dtype == PA_KV_FP16) hipLaunchKernelGGL((keep_rows_kernel<2>), both, block, 0, s, a);
    else if (dtype == PA_KV_FP8_E4M3) hipLaunchKernelGGL((keep_rows_kernel<1>), both, block, 0, s, a);
    else hipLaunchKernelGGL(keep_blocks_kernel, grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace pa
