// gfx950 attention of several new tokens per sequence over a paged cache: drafted
// trees, chains, pieces of prompts. (No counterpart in the reference.)
//
//   tree_attention_kernel   the work, in equal shares
//   tree_merge_kernel       tiles that shares cut apart, joined; values that are not finite
//
// out_i = sum_p exp(s_ip - m_i) v_p / sum_p exp(s_ip - m_i), s_ip = sm_scale q_i k_p, over the
// places p that token i sees: one pass with a running m_i, sums in 32 bits.
//
// Rows and tiles. The query heads of a kv head and the tokens of an entry are rows of one
// product, token by token, so a place is read once for all of them: tiles of 64, 128 or 256
// rows, 32 a wave. A tile walks its places in steps of 64 to 128 (kStep). Waves of one tile share
// a stream of places (WQ of them); WK streams take a part of every step each and are joined at the end.
//
// Shares. Lengths are device data, so the host cannot lay out the work: every block adds up the
// entries' costs and takes one of gridDim.x equal shares of (entry, kv head, tile, step), in that
// order. A share cuts at most two tiles, whose sums go to the workspace (two slots a block). One
// token over 131072 places and a prompt of 4096 go through the same code.
//
// Products. S^T = K Q^T with v_mfma_f32_32x32x16_f16: a lane holds 16 places of one row, so the
// softmax needs one exchange between the wave's halves, and P^T is the second product's operand
// as it lies. O^T = V^T P^T, V's fragments read transposed from LDS (ds_read_b64_tr_b16). K and V
// go through registers into LDS as fp16: FP8 is widened once for all of the tile's rows, a block's
// scale of V along with it (within 2^-25, as the decode has it), and places that are not there become
// zeros. K's goes into its scores in 32 bits (345 / 357 us for 32 tokens over 64 x 8192 with K scaled
// in fp16 and so, but fp16 has no keys below 2^-24). Two buffers, loads a whole step ahead.
//
// What bounds it (one MI355X): trees of few rows, memory (1 token over 32 x 8192, fp16: 170 us,
// 6.3 TB/s; 16: 168); tiles of 128 rows and more, three pipes: 32 places by 32 rows are 16 MFMAs of
// 32 cycles, per lane 16 exponentials, maxima, sums and roundings besides the staging, and 16 KB out
// of LDS, which a wave reads for its 32 rows alone (45% of its time at 128 bytes a cycle; its counter
// says 29%). The matrix pipe is busy 45% of the time, the vector pipe 43%, and no order of the code that was
// tried laid them wholly over each other (4096 tokens after 4096: 458 to 474 us, 870 to 900 TFLOP/s, a large
// library product 1232; 32 over 64 x 8192, block scales: 357 to 371). Twice the rows a wave, half the
// reads, does not fit the registers (705 us, 130 spilled). Small calls: the instructions of a tile's
// prologue and end, and the merge's launch (8 tokens over 200: 11 us, 3 of them the merge's).

#include "pa_device.hpp"
#include "pa_fp8.hpp"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace pa {
namespace {

typedef float    f32x16 __attribute__((ext_vector_type(16)));
typedef float    f32x2  __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2  __attribute__((ext_vector_type(2)));
typedef short    s16x4  __attribute__((ext_vector_type(4)));

constexpr int kSub     = 32;              // places of one MFMA step
constexpr int kScan    = 256;             // entries that a block looks at together
constexpr int kMergeWaves = 4, kMergeRows = 2 * kMergeWaves;
constexpr int kItemUnits  = 3;   // what a tile costs besides its steps, in steps
constexpr int kMinStep    = 64;  // places of a step, at least
// Entries with more units than this are left out, all of them (divide() takes less than 2^53). Entries
// that lie behind one another have fewer: at most kMaxTreeRows tiles, as a tile and kv head has a row of
// its own at least, and a tile kItemUnits, its steps over 2^31 places at most, one for rounding and, in
// a chain, one more.
constexpr long kMaxUnits  = (1l << 53) - (1l << 20);
static_assert(kMaxTreeRows * (kItemUnits + 2 + (1l << 31) / kMinStep) <= kMaxUnits);
constexpr int kSchedMfma = 0x8, kSchedLds = 0x100;   // of sched_group_barrier
constexpr int kDesc    = 8;               // ints of a block's entry for the merge: parts, first token, tokens, kv head, 8 bytes of odd_flag
constexpr int kOutLd   = kHeadDim + 4;    // floats of a row in the joining of waves

// A probability is kept as 2^(score - reference + kShift) in fp16, where the reference
// follows the row's maximum with a lag of at most kLag: 2^14 at most, and normal down
// to 2^-20 of the maximum (fp16 is subnormal below 2^-14).
constexpr float kShift = 6.0f;
constexpr float kLag   = 8.0f;

// Accesses to global memory through pointers that come from memory (arguments() below): without
// saying where they point, they count as LDS accesses, too, and out of order, and
// every wait for a fragment then waits for all of them.
template <class T>
using Global = __attribute__((address_space(1))) T;
template <class T>
__device__ __forceinline__ T load_global(const void* p) {
    return *(const Global<T>*)(p);
}
template <class T>
__device__ __forceinline__ void store_global(void* p, T x) {
    *(Global<T>*)(p) = x;
}

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
                    static_cast<long>(x.start) + x.n <= min(static_cast<long>(c.table_stride) * c.page_size, static_cast<long>(INT_MAX - 256));
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
                    static_cast<long>(x.start) + x.n <= min(static_cast<long>(c.table_stride) * c.page_size, static_cast<long>(INT_MAX - 256));
    if (!ok) x.n = 0;
    return x;
}

// Units of work of the first j row tiles of an entry and one kv head: their steps over the places
// that they are given, and kItemUnits each for what a tile costs besides (its queries, the first
// rows' way through the page table, its output: 7 to 10 us, a step of 256 rows 3.5). us with 0, 1, 2,
// 3 and 5: 1 to 60 tokens after 37 ragged sequences 178, 146, 130, 124, 128; with 2, 3, 4 and 6: 4096
// tokens after 4096 460, 464, 478, 482, 8 after 37 ragged ones 47, 45, 44, 46. For a tree j
// times the steps over all of the entry's places; for a chain, whose tile i ends at place start +
// (i + 1) tile_tokens, the sum of these ends over the step, and one more a tile, which covers what
// rounding up adds.
__device__ __forceinline__ long steps_before(const TreeAttention& a, const Entry& x, int step, int j) {
    if (a.tree) return static_cast<long>(j) * (kItemUnits + (x.start + x.n + step - 1) / step);
    return static_cast<long>(j) * (kItemUnits + 1) + (static_cast<long>(j) * x.start + static_cast<long>(j) * (j + 1) / 2 * a.tile_tokens) / step;
}
__device__ __forceinline__ int tiles_of(const TreeAttention& a, const Entry& x) { return a.by_tile.of(x.n + a.tile_tokens - 1); }
__device__ __forceinline__ long entry_cost(const TreeAttention& a, const Entry& x, int step) {
    return x.n == 0 ? 0 : steps_before(a, x, step, tiles_of(a, x)) * a.c.hkv;
}

// The kernel's arguments, read again where this is called: read once, at the kernel's start, the
// seventy scalars would be held (and spilled) through everything.
__device__ __forceinline__ TreeAttention arguments() {
    using words = const __attribute__((address_space(4))) uint32_t*;
    words p = (words)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    uint32_t w[sizeof(TreeAttention) / 4];
#pragma unroll
    for (size_t i = 0; i < sizeof(TreeAttention) / 4; ++i) w[i] = p[i];
    TreeAttention a;
    __builtin_memcpy(&a, w, sizeof a);
    return a;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// A value that every lane has the same, as a scalar (what comes from LDS or a shuffle is
// taken to differ, and then so is every loop that it bounds).
__device__ __forceinline__ long uniform(long x) {
    return static_cast<long>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32)))) << 32 |
                             static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))));
}

// a / b for 0 <= a < 2^53, 0 < b, wave-uniform: in 32 bits where a is small (nearly always), else
// through doubles (a 64-bit integer division is 140 scalar instructions). Either quotient is off
// by one at most before it is put right.
__device__ __forceinline__ long divide(long a, long b) {
    if (a < (1 << 22)) {
        if (b > a) return 0;
        const int x = static_cast<int>(a), y = static_cast<int>(b);
        int q = static_cast<int>(static_cast<float>(x) * __builtin_amdgcn_rcpf(static_cast<float>(y)));
        const int r = x - q * y;
        q += r >= y ? 1 : r < 0 ? -1 : 0;
        return uniform(q);
    }
    long q = static_cast<long>(static_cast<double>(a) / static_cast<double>(b));
    const long r = a - q * b;
    q += r >= b ? 1 : r < 0 ? -1 : 0;
    return uniform(q);
}

struct Schedule {
    long pre[kScan + 1];   // units before each entry of the chunk
    long wave_sum[kScan / 64];
    int  hit;
};

// The units of entries c0 .. c0 + 255 as a running sum in s.pre (by the block's first 256 threads).
__device__ __forceinline__ long scan_chunk(const TreeAttention& a, Schedule& s, int c0, int step) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.c.n_ent == 1) return entry_cost(a, entry_at(a.c, 0), step);   // nothing to look for
    const bool mine = tid < kScan;
    long x = mine && c0 + tid < a.c.n_ent ? entry_cost(a, entry_of_lane(a.c, c0 + tid), step) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (mine && lane == 63) s.wave_sum[wave] = x;
    __syncthreads();
    long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kScan / 64; ++w) {
        if (w < wave) before += s.wave_sum[w];
        total += s.wave_sum[w];
    }
    if (mine) s.pre[tid + 1] = before + x;
    if (tid == 0) s.pre[0] = 0;
    __syncthreads();
    return uniform(total);
}

// A part of a share: units u0 .. u1 - 1 of a tile's `units` (more than kItemUnits at least), the first of them unit w of the call.
struct Share {
    Entry x;
    int   h, rt, u0, u1, units;
    long  w, per;
};

// f(share) for what block lb of nb has to do, in order. (All threads of a block of 256 at least.)
template <class F>
__device__ __forceinline__ void walk(const TreeAttention& a, Schedule& sch, int nb, int lb, int step, F&& f) {
    long total = 0, chunk = 0;
    for (int c0 = 0; c0 < a.c.n_ent && total <= kMaxUnits; c0 += kScan) total += chunk = scan_chunk(a, sch, c0, step);
    if (total > kMaxUnits) total = 0;
    const long per = max(divide(total + nb - 1, nb), 1l);
    long w = lb * per;
    const long w_end = min(w + per, total);
    if (w >= w_end) return;
    int  c0 = 0;
    long before = 0;
    if (a.c.n_ent > kScan) chunk = scan_chunk(a, sch, 0, step);
    while (w < w_end) {
        while (w >= before + chunk) {
            before += chunk;
            c0 += kScan;
            if (c0 >= a.c.n_ent) return;   // (the entries were changed under the call, here and below)
            chunk = scan_chunk(a, sch, c0, step);
        }
        int  hit = 0;
        long at  = 0;
        if (a.c.n_ent > 1) {
            const int tid = threadIdx.x;
            if (tid < kScan && sch.pre[tid] <= w - before && w - before < sch.pre[tid + 1]) sch.hit = tid;
            __syncthreads();
            hit = min(max(__builtin_amdgcn_readfirstlane(sch.hit), 0), min(kScan, a.c.n_ent - c0) - 1);
            at  = before + uniform(sch.pre[hit]);
            __syncthreads();
        }
        Share s;
        s.x   = entry_at(a.c, c0 + hit);
        s.x.n = uniform(s.x.n);
        if (s.x.n == 0) return;
        const int  tiles = tiles_of(a, s.x);
        const long head_steps = uniform(steps_before(a, s.x, step, tiles));
        const long local = w - at;
        s.h = static_cast<int>(divide(local, head_steps));
        const long inner = local - s.h * head_steps;
        if (s.h < 0 || s.h >= a.c.hkv || inner < 0) return;
        int rt = 0;   // the last tile that begins at or before
        for (int span = tiles; span > 1;) {
            const int half = span / 2;
            if (steps_before(a, s.x, step, rt + half) <= inner) rt += half;
            span -= half;
        }
        s.rt = uniform(rt);
        const long first = uniform(steps_before(a, s.x, step, s.rt));
        s.units = static_cast<int>(uniform(steps_before(a, s.x, step, s.rt + 1)) - first);
        s.u0 = static_cast<int>(inner - first);
        s.u1 = static_cast<int>(min(static_cast<long>(s.units), s.u0 + (w_end - w)));
        s.w  = w;
        s.per = per;
        // A tile's first kItemUnits are no steps: a share that ends among them leaves the tile to the next block.
        if (s.u1 > kItemUnits) f(s);
        w += max(s.u1 - s.u0, 1);   // (1 as above; a return here slows the long loops by 3%)
    }
}

// Whether wave w of block lb met values that are not finite.
__device__ __forceinline__ uint8_t* odd_flag(int32_t* desc, int lb, int w) { return reinterpret_cast<uint8_t*>(desc + kDesc * lb + 4) + w; }

// Bytes of a staged row: 128 fp16 and some more, so that the rows that a fragment read takes at
// once lie in different banks (64 of 4 bytes: 16 rows of K, 16 bytes of each; 4 rows of V, 64
// bytes of each), and every fragment at a constant distance from the lane's first.
constexpr int kRowK = 256 + 16, kRowV = 256 + 64;

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
        if (j0 > -32) bits |= static_cast<uint32_t>(load_global<uint64_t>(row) << -j0);
    } else {
        const int w = j0 >> 6, sh = j0 & 63;
        uint64_t v = w < a.words ? load_global<uint64_t>(row + w) >> sh : 0;
        if (sh > 32 && w + 1 < a.words) v |= load_global<uint64_t>(row + w + 1) << (64 - sh);
        bits = static_cast<uint32_t>(v);
    }
    return bits & ones(x.n - j0);
}

// EB: bytes of a cached value; BS: block scales. A wave holds 32 rows of queries; WQ
// waves of rows share a stream of places, WK streams are joined at the end. UNI: pages
// hold whole runs of 4 places, so a load of 4 rows lies in one page.
template <int EB, bool BS, int WQ, int WK, bool UNI>
struct TreeKernel {
    static constexpr int kWaves  = WQ * WK;
    static constexpr int kBlock  = 64 * kWaves;
    static constexpr int kRowsM  = 32 * WQ;
    static constexpr int SUBS    = WQ >= 4 ? 2 : 1;            // 32-place parts of a stream's step
    static constexpr int HALVES  = WQ == 8 && UNI ? 2 : 1;     // turns of that many parts between two barriers
    static constexpr int kTurn   = kSub * SUBS;
    static constexpr int kPart   = kTurn * HALVES;             // places of a stream's step
    static constexpr int kStep   = kPart * WK;
    static constexpr int NJ      = kPart / (4 * WQ);           // loads of 4 rows per wave, of K and of V
    static constexpr int kTileK  = kPart * kRowK, kTileV = kPart * kRowV;   // bytes of a step's rows
    static constexpr int kBuf    = kTileK + kTileV;
    static constexpr int kStage  = WK * 2 * kBuf;
    static constexpr int kJoin   = kWaves * 32 * (kOutLd * 4 + 8);
    static constexpr int kLds    = kStage > kJoin ? kStage : kJoin;
    // Loads bypass the caches where hardly any place is read twice: tiles of 64 and 128 rows, which hold all of an
    // average entry's. (us with cached and with such loads: 16 over 32 x 8192 fp16 219 / 203, 4096 over 4096 451 / 511.
    // An entry of many tiles beside short ones that make the call's tiles small has its places read past the caches, too.)
    static constexpr int kAux    = WQ < 8 ? 2 : 0;
    static constexpr int RG      = UNI ? 4 : 1;                // rows that a lane looks up
    static_assert(kPart / RG <= 64 && NJ >= 1 && kStep >= kMinStep);

    typedef uint32_t Raw __attribute__((ext_vector_type(EB == 2 ? 4 : 2)));

    static __device__ __forceinline__ void run(const TreeAttention& a, unsigned char* lds, Schedule& sch) {
        // The block's share of the units, consecutive ones on one XCD (blocks go round the 8 XCDs).
        const int nb = gridDim.x;
        const int lb = nb % 8 == 0 ? (blockIdx.x % 8) * (nb / 8) + blockIdx.x / 8 : blockIdx.x;
        int32_t* const desc = a.desc + kDesc * lb;   // what the merge has to do from here on
        if (threadIdx.x == 0) desc[0] = 1;
        if (threadIdx.x % 64 == 0)
            for (int w = threadIdx.x / 64; w < 8; w += kWaves) store_global<uint8_t>(odd_flag(a.desc, lb, w), 0);
        walk(a, sch, nb, lb, kStep, [&](const Share& s) __attribute__((always_inline)) {
            const Entry& x = s.x;
            const bool begins = s.u0 <= kItemUnits, ends = s.u1 == s.units;
            if (begins && !ends && threadIdx.x == 0) {   // the block's last tile: its other parts are the next blocks' first
                desc[1] = x.t0 + s.rt * a.tile_tokens;
                desc[2] = min(a.tile_tokens, x.n - s.rt * a.tile_tokens);
                desc[3] = s.h;
                desc[0] = static_cast<int>(divide(s.w - s.u0 + s.units - 1, s.per)) - lb + 1;
            }
            item_part(lds, x, s.h, s.rt, uniform(max(s.u0, kItemUnits) - kItemUnits), uniform(s.u1 - kItemUnits),
                      uniform(begins && ends ? -1 : 2 * lb + (begins ? 1 : 0)), lb);
        });
    }

    static __device__ __forceinline__ void item_part(unsigned char* lds, const Entry& x, int h, int rt, int k0,
                                                     int k1, int slot, int lb) {
        const TreeAttention a = arguments();
        const CachedTokens& c = a.c;
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave % WQ, wk = wave / WQ;
        const int ql = lane & 31, hl = lane >> 5;
        const int G = a.group, P = c.page_size;
        const int tok0 = rt * a.tile_tokens;   // first token of the tile, within the entry
        const int tile_n = uniform(min(a.tile_tokens, x.n - tok0));
        const int end = uniform(x.start + (a.tree ? x.n : tok0 + tile_n));   // places from here on are not seen
        k1 = uniform(min(k1, (end + kStep - 1) / kStep));

        const bool has_rows = 32 * wq < tile_n * G;   // else the wave only stages
        const int all_open = uniform(x.start + (a.tree ? 0 : tok0 + 1));   // places before this one are seen by every row

        f32x16 o[4];
        float  m = -INFINITY, l = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

        // Staging. Lane i looks up rows RG i .. of a step; load j of a wave takes the 4 rows
        // from 4 (wq + WQ j) on, 16 lanes a row, 8 dims each.
        const int row0 = lane >> 4, ch = lane & 15;
        const int32_t* table = c.table + static_cast<size_t>(x.row) * c.table_stride;
        const size_t page_bytes = static_cast<size_t>(c.hkv) * P * kRowBytes<EB>;
        const size_t head_off   = static_cast<size_t>(h) * P * kRowBytes<EB>;
        const int    bsh = BS ? (P % 16 == 0 ? 4 : 3) : 0, nblk = BS ? P >> bsh : 0;
        int      pg = -1;
        Raw      kr[NJ], vr[NJ];
        uint32_t sc = 0;       // the lane's rows' scale pair
        float    k_sc = 0.f;   // of the step in the stage: the scale of K's scores, into base-2 exponents
        uint32_t live = 0;     // general pages: loads whose row holds a place
        auto lookup = [&](int k) {
            const int t = k * kStep + kPart * wk + RG * lane;
            pg = lane < kPart / RG && t < end ? load_global<int32_t>(table + a.by_page.of(t)) : -1;
        };
        if (k0 < k1) lookup(k0);   // (before the queries' loads, which come back in order)

        // The tile's queries, 16 lanes a row, on their way to LDS (loaded as fragments, each load would
        // touch 32 lines: 4 us an item with 8 waves). A negative scale turns their signs.
        const float    score_scale = fmaxf(fabsf(a.score_scale), FLT_MIN);   // (of 0, one that makes every score 0 but minus infinity)
        const uint32_t flip = a.score_scale < 0.f ? 0x80008000u : 0u;
        constexpr int NQ = kRowsM * 16 / kBlock;
        f16x8 q[8];
        u32x4 qr[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int row = (tid >> 4) + j * (kBlock / 16), i = a.by_group.of(row), g = row - i * G;
            const bool ok = i < tile_n;
            qr[j] = load_global<u32x4>(a.q + (x.t0 + tok0 + (ok ? i : 0)) * a.q_stride + (h * G + (ok ? g : 0)) * kHeadDim + 8 * (tid & 15));
        }
        const int my_row = 32 * wq + ql, my_i = a.by_group.of(my_row);
        const int tok = my_i < tile_n ? tok0 + my_i : INT_MAX;
        auto issue = [&](int k) {
            const int  t  = k * kStep + kPart * wk + RG * lane;
            const bool ok = pg >= 0 && pg < c.num_pages;
            const int  s  = t - a.by_page.of(t) * P;
            const size_t off = ok ? pg * page_bytes + head_off + static_cast<size_t>(s) * kRowBytes<EB> : 0;
            const uint32_t lo = static_cast<uint32_t>(off), hi = static_cast<uint32_t>(off >> 32);
            const int rows = ok ? min(RG, end - t) : 0;
            if constexpr (BS)
                sc = rows > 0 ? load_global<uint16_t>(c.scales + 2 * ((static_cast<size_t>(pg) * c.hkv + h) * nblk + (s >> bsh))) : 0;
            live = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int r4 = wq + WQ * j;   // run of 4 rows
                if constexpr (UNI) {
                    const size_t at = static_cast<size_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, r4))) << 32 |
                                      static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, r4));
                    const int bytes = __builtin_amdgcn_readlane(rows, r4) * kRowBytes<EB>;
                    const __amdgpu_buffer_rsrc_t kb = buffer_rsrc(static_cast<const unsigned char*>(c.k_cache) + at, bytes);
                    const __amdgpu_buffer_rsrc_t vb = buffer_rsrc(static_cast<const unsigned char*>(c.v_cache) + at, bytes);
                    if constexpr (EB == 2) {
                        kr[j] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(kb, 16 * lane, 0, kAux));
                        vr[j] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(vb, 16 * lane, 0, kAux));
                    } else {
                        kr[j] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(kb, 8 * lane, 0, kAux));
                        vr[j] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(vb, 8 * lane, 0, kAux));
                    }
                } else {
                    const int from = 4 * r4 + row0;
                    const size_t at = (static_cast<size_t>(static_cast<uint32_t>(__shfl(static_cast<int>(hi), from))) << 32 |
                                       static_cast<uint32_t>(__shfl(static_cast<int>(lo), from))) + ch * 8 * EB;
                    live |= __shfl(rows, from) > 0 ? 1u << j : 0u;
                    kr[j] = load_global<Raw>(static_cast<const unsigned char*>(c.k_cache) + at);
                    vr[j] = load_global<Raw>(static_cast<const unsigned char*>(c.v_cache) + at);
                }
            }
        };
        auto widen = [](Raw x, float scale) {
            if constexpr (EB == 2) return x;
            else return u32x4{fp8x2_to_f16x2<false>(x[0], scale), fp8x2_to_f16x2<true>(x[0], scale),
                              fp8x2_to_f16x2<false>(x[1], scale), fp8x2_to_f16x2<true>(x[1], scale)};
        };
        auto stage_at = [&](int buf) { return lds + (2 * wk + buf) * kBuf; };
        // A place that a row does not see must not reach it, whatever its value: 0 * infinity is
        // NaN. So where rows see different places (masked), values that are not finite are staged as
        // zeros; the merge has them at the end (odd_tile).
        auto tell = [&] {
            if (lane == 0) store_global<uint8_t>(odd_flag(arguments().desc, lb, wave), 1);
        };
        auto store = [&](int buf, auto masked_c) {
            constexpr bool masked = decltype(masked_c)::value;
            unsigned char* k = stage_at(buf);
            u16x2 largest = {0, 0};
            // (In 32 bits: under its smallest scales K is below what fp16 holds, at its largest past it. Within the
            // positive normal numbers, so that minus infinity stays what it is and 0 stays 0.)
            if constexpr (BS) k_sc = fminf(fmaxf(score_scale * __builtin_bit_cast(float, (sc & 0xff) << 23), FLT_MIN), FLT_MAX);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int r4 = wq + WQ * j, row = 4 * r4 + row0;
                float vs = 1.0f;   // (the conversion takes V's scale along)
                if constexpr (BS) vs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(sc, r4 * 4 / RG) >> 8 << 23);
                u32x4 kx = widen(kr[j], 1.0f), vx = widen(vr[j], vs);
                if (!UNI && !(live >> j & 1)) kx = vx = u32x4{0, 0, 0, 0};
                *reinterpret_cast<u32x4*>(k + row * kRowK + 16 * ch) = kx;
                if constexpr (masked) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, vx[e] & 0x7fff7fffu));
                }
                *reinterpret_cast<u32x4*>(k + kTileK + row * kRowV + 16 * ch) = vx;
            }
            if constexpr (masked) {
                const bool any = __builtin_amdgcn_ballot_w64(largest[0] >= 0x7c00 || largest[1] >= 0x7c00) != 0;
                if (any) {
                    tell();
#pragma unroll 1
                    for (int j = 0; j < NJ; ++j) {   // (a lane's own values, again)
                        u32x4* const at = reinterpret_cast<u32x4*>(k + kTileK + (4 * (wq + WQ * j) + row0) * kRowV + 16 * ch);
                        u32x4 vx = *at;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((vx[e] & 0x7c00u) == 0x7c00u) vx[e] &= 0xffff0000u;
                            if ((vx[e] & 0x7c000000u) == 0x7c000000u) vx[e] &= 0xffffu;
                        }
                        *at = vx;
                    }
                }
            }
        };
        // Where this lane's fragments of V lie in the stage.
        const int va = (4 * hl + ((lane & 15) >> 2)) * kRowV + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

        auto step_of = [&](auto masked_c, int base, const unsigned char* buf, int turn) {
            constexpr bool MASK = decltype(masked_c)::value;
            // And of K, worked out in every step: held, it would be spilled, and a wait for a spilled
            // register is one for the loads of the next step, too (1% of a chain of 4096).
            unsigned all = ~0u;
            asm volatile("" : "+s"(all));
            const int self = __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0));
            const int ka = (self & 31) * kRowK + 16 * (self >> 5);
            const unsigned char* ks = buf + turn * kTurn * kRowK;
            const unsigned char* vs = buf + kTileK + turn * kTurn * kRowV;
            auto k_frag = [&](int n) {   // of part n % SUBS, dims 16 (n / SUBS) .. (the parts' sums in turn)
                return *reinterpret_cast<const f16x8*>(ks + ka + 32 * (n / SUBS) + n % SUBS * kSub * kRowK);
            };
            auto v_part = [&](int n, int w) {
                const int at = va + 64 * (n % 4) + (16 * (n / 4) + 8 * w) * kRowV;
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vs + at));
            };
            auto v_frag = [&](int n) {   // of 16 places from 16 (n / 4) on, dims 32 (n % 4) ..
                const s16x4 lo = v_part(n, 0), hi = v_part(n, 1);
                return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            // Fragments are read eight products ahead; the first of V before the softmax.
            f32x16 s[SUBS];
            f16x8  kf[8], vf[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) kf[n] = k_frag(n);
#pragma unroll
            for (int b = 0; b < SUBS; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
            for (int n = 0; n < 8 * SUBS; ++n) {
                s[n % SUBS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n % 8], q[n / SUBS], s[n % SUBS], 0, 0, 0);
                if (n + 8 < 8 * SUBS) kf[n % 8] = k_frag(n + 8);
                else vf[n % 8] = v_frag(n % 8);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedLds, 8, 0);
#pragma unroll
            for (int n = 0; n < 8 * (SUBS - 1); ++n) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedLds, 1, 0);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedLds, 2, 0);
            }
            uint32_t seen[SUBS];
            float top = -INFINITY, cs[SUBS][4];   // scales of scores: a block has 8 places or 16
#pragma unroll
            for (int b = 0; b < SUBS; ++b) {
#pragma unroll
                for (int i = 0; i < 4; ++i) cs[b][i] = BS ? readlane_f(k_sc, (kTurn * turn + kSub * b + 8 * i) / RG) : score_scale;
                if constexpr (MASK) {
                    seen[b] = visible(a, x, tok, base + kSub * b - x.start);
                    const uint32_t mine = seen[b] >> (4 * hl);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        // (By bits: a comparison each would hold 16 lane masks at once.)
                        const uint32_t all = __builtin_amdgcn_sbfe(mine, 8 * (i / 4) + i % 4, 1);
                        const float    raw = s[b][i];
                        const uint32_t y = __builtin_bit_cast(uint32_t, raw) & all;
                        s[b][i] = __builtin_bit_cast(float, y | (~all & 0xff800000u));
                    }
                }
                if constexpr (BS) {   // (scales are above 0)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float t = -INFINITY;   // (from the values alone, two would be made canonical first)
#pragma unroll
                        for (int e = 0; e < 4; ++e) t = fmaxf(t, s[b][i + e]);
                        top = fmaxf(top, t * cs[b][i / 4]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
                }
            }
            top = max_halves(top);
            if constexpr (!BS) top *= score_scale;   // (which is not below 0)
            if (__builtin_amdgcn_ballot_w64(top > m + kLag) != 0) {
                const float now = fmaxf(m, top), ref = now == -INFINITY ? 0.f : now;
                const float f = exp2_fast(m - ref);
                l *= f;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= f;
                m = now;
            }
            const float ref = (m == -INFINITY ? 0.f : m) - kShift;
            const f16x2 ones2 = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
            f16x8 p[SUBS][2];
#pragma unroll
            for (int b = 0; b < SUBS; ++b)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float e0 = exp2_fast(fmaf(s[b][i], cs[b][i / 4], -ref));
                    const float e1 = exp2_fast(fmaf(s[b][i + 1], cs[b][i / 4], -ref));
                    // (Summed as they are rounded, two an instruction, in 32 bits.)
                    const f16x2 e = {static_cast<_Float16>(e0), static_cast<_Float16>(e1)};
                    l = __builtin_amdgcn_fdot2(e, ones2, l, false);
                    p[b][i / 8][i % 8] = e[0];
                    p[b][i / 8][i % 8 + 1] = e[1];
                }
#pragma unroll
            for (int n = 0; n < 8 * SUBS; ++n) {
                o[n % 4] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n % 8], p[n / 8][n / 4 % 2], o[n % 4], 0, 0, 0);
                if (n + 8 < 8 * SUBS) vf[n % 8] = v_frag(n + 8);
            }
            if constexpr (SUBS == 2) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 1);
                    __builtin_amdgcn_sched_group_barrier(kSchedLds, 2, 1);
                }
            }
        };

        if (k0 < k1) {
            issue(k0);
            if (k0 + 1 < k1) lookup(k0 + 1);
        }
        // (At the end of the stage: in the last buffer where they fit there, which the first step does not write.)
        unsigned char* const qs = lds + kStage - kRowsM * kRowK;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) qr[j][e] ^= flip;
            *reinterpret_cast<u32x4*>(qs + ((tid >> 4) + j * (kBlock / 16)) * kRowK + 16 * (tid & 15)) = qr[j];
        }
        block_sync();
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s] = *reinterpret_cast<const f16x8*>(qs + my_row * kRowK + 32 * s + 16 * hl);
        if constexpr (kRowsM * kRowK > kBuf) block_sync();
        // Steps that every row sees whole, then those that rows see in part: two loops, so that the
        // second's masks cost the first neither registers nor copies of the sums.
        auto steps = [&](auto masked_c, int from, int to) {
            constexpr bool MASK = decltype(masked_c)::value;
#pragma unroll 1
            for (int k = from; k < to; ++k) {
                const int buf = (k - k0) & 1;
                const int base = k * kStep + kPart * wk;
                store(buf, masked_c);
                if (k + 1 < k1) {
                    issue(k + 1);
                    if (k + 2 < k1) lookup(k + 2);
                }
                block_sync();
                if (has_rows) {
#pragma unroll
                    for (int t = 0; t < HALVES; ++t)
                        if (!MASK || base + kTurn * t < end) step_of(masked_c, base + kTurn * t, stage_at(buf), t);
                }
            }
        };
        const int mid = uniform(max(k0, min(k1, all_open / kStep)));
        steps(std::false_type{}, k0, mid);
        steps(std::true_type{}, mid, k1);

        const float sum = add_halves(l);
        if constexpr (WK == 1) {
            // The wave has its rows' whole sums. They go through LDS, so that a store takes whole rows.
            float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) zero[d] = fmaf(o[d][i], 0.f, zero[d]);
            // (NaN is not 0. Sums that are not finite, of rows whose softmax is, come of values in steps without masks.)
            if (__builtin_amdgcn_ballot_w64((zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.f && sum == sum) != 0) tell();
            block_sync();   // no wave reads the stage any more
            unsigned char* const mine = lds + wave * 32 * kOutLd * 4;
            if (slot >= 0) {
                const size_t at = static_cast<size_t>(slot) * kRowsM + 32 * wq;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4*>(mine + 4 * (ql * kOutLd + 32 * d + 8 * i + 4 * hl)) =
                            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                wave_lds_sync();
                if (hl == 0) store_global(a.part_ml + 2 * (at + ql), f32x2{m, sum});
#pragma unroll 4
                for (int r = 0; r < 32; r += 2)
                    store_global(a.part_out + (at + r + hl) * kHeadDim + 4 * ql,
                                 *reinterpret_cast<const f32x4*>(mine + 4 * ((r + hl) * kOutLd + 4 * ql)));
            } else if (has_rows) {
                const float scale = sum == 0.f ? 0.f : c.v_scale / sum;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f16x2 lo = {static_cast<_Float16>(o[d][4 * i] * scale), static_cast<_Float16>(o[d][4 * i + 1] * scale)};
                        const f16x2 hi = {static_cast<_Float16>(o[d][4 * i + 2] * scale), static_cast<_Float16>(o[d][4 * i + 3] * scale)};
                        *reinterpret_cast<u32x2*>(mine + ql * kRowK + 64 * d + 16 * i + 8 * hl) =
                            u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
                    }
                wave_lds_sync();
#pragma unroll 4
                for (int r = lane >> 4; r < 32; r += 4) {
                    const int i = a.by_group.of(32 * wq + r), g = 32 * wq + r - i * G;
                    if (i < tile_n)
                        store_global(a.out + (x.t0 + tok0 + i) * a.out_stride + (h * G + g) * kHeadDim + 8 * (lane & 15),
                                     *reinterpret_cast<const u32x4*>(mine + r * kRowK + 16 * (lane & 15)));
                }
            }
            block_sync();   // the stage is free again
            return;
        }

        // The streams joined through LDS.
        float* const ol = reinterpret_cast<float*>(lds);
        float* const ml = ol + kWaves * 32 * kOutLd;
        __syncthreads();
        float* mine = ol + (32 * wave + ql) * kOutLd;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(mine + 32 * d + 8 * i + 4 * hl) =
                    f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (hl == 0) *reinterpret_cast<f32x2*>(ml + 2 * (32 * wave + ql)) = f32x2{m, sum};
        __syncthreads();
        constexpr int TR = kBlock / kRowsM;   // threads of a row
        const int row = tid / TR, part = tid % TR;
        float top = -INFINITY, den = 0.f, f[WK];
#pragma unroll
        for (int g = 0; g < WK; ++g)
            top = fmaxf(top, ml[2 * (kRowsM * g + row)]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int g = 0; g < WK; ++g) {
            const float* e = ml + 2 * (kRowsM * g + row);
            f[g] = exp2_fast(e[0] - ref);
            den += f[g] * e[1];
        }
        const int i = a.by_group.of(row), g0 = row - i * G;
        float zero = 0.f;
        if (i < tile_n) {
            const float scale = slot >= 0 ? 1.f : den == 0.f ? 0.f : c.v_scale / den;
            uint16_t* out = a.out + (x.t0 + tok0 + i) * a.out_stride + (h * G + g0) * kHeadDim;
            const size_t at = static_cast<size_t>(max(slot, 0)) * kRowsM + row;
#pragma unroll
            for (int n = 0; n < 32 / TR; ++n) {
                const int d = 4 * (part + TR * n);
                f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < WK; ++g) {
                    const f32x4 z = *reinterpret_cast<const f32x4*>(ol + (kRowsM * g + row) * kOutLd + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = fmaf(z[e], f[g], y[e]);
                }
                zero = fmaf(y[0], 0.f, fmaf(y[1], 0.f, fmaf(y[2], 0.f, fmaf(y[3], 0.f, zero))));
                if (slot >= 0) {
                    store_global(a.part_out + at * kHeadDim + d, y);
                } else {
                    const f16x2 lo = {static_cast<_Float16>(y[0] * scale), static_cast<_Float16>(y[1] * scale)};
                    const f16x2 hi = {static_cast<_Float16>(y[2] * scale), static_cast<_Float16>(y[3] * scale)};
                    store_global(out + d, u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)});
                }
            }
            if (slot >= 0 && part == 0) store_global(a.part_ml + 2 * at, f32x2{top, den});
        }
        if (__builtin_amdgcn_ballot_w64(zero != 0.f && den == den) != 0) tell();   // (as above)
        __syncthreads();   // the stage is free again
    }
};

template <int EB, bool BS, int WQ, int WK, bool UNI>
__global__ __launch_bounds__(64 * WQ * WK, 2) void tree_attention_kernel(const TreeAttention a) {
    using T = TreeKernel<EB, BS, WQ, WK, UNI>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[T::kLds];
    __shared__ Schedule sch;
    T::run(a, lds, sch);
}

// A row's n parts joined by half a wave, a lane four sums; U parts are on their way.
template <int U>
__device__ __forceinline__ void merge_row(const TreeAttention& a, int n, int block, int row, int t, int head) {
    const int d4 = 4 * (threadIdx.x & 31);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, den = 0.f;
    for (int k0 = 0; k0 < n; k0 += U) {
        f32x2 e[U];
        f32x4 y[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int    part = min(k0 + k, n - 1);
            const size_t at = static_cast<size_t>(2 * (block + part) + (part == 0)) * a.rows + row;
            e[k] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * at);
            y[k] = *reinterpret_cast<const f32x4*>(a.part_out + at * kHeadDim + d4);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const bool  mine = k0 + k < n;
            const float lse = mine ? e[k][0] : -INFINITY, now = fmaxf(m, lse), ref = now == -INFINITY ? 0.f : now;
            const float f0 = exp2_fast(m - ref), f1 = exp2_fast(lse - ref);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = acc[c] * f0 + (mine ? y[k][c] : 0.f) * f1;
            den = den * f0 + (mine ? e[k][1] : 0.f) * f1;
            m = now;
        }
    }
    const float scale = den == 0.f ? 0.f : a.c.v_scale / den;
    const f16x2 lo = {static_cast<_Float16>(acc[0] * scale), static_cast<_Float16>(acc[1] * scale)};
    const f16x2 hi = {static_cast<_Float16>(acc[2] * scale), static_cast<_Float16>(acc[3] * scale)};
    *reinterpret_cast<u32x2*>(a.out + t * a.out_stride + head * kHeadDim + d4) =
        u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// Values that are not finite into a tile's result, kMergeRows rows of it, half a wave each: a token that sees
// one has it in that dim, of whatever weight. (A weight that is 0 in fp16, or in 32 bits, makes NaN of an
// infinity, and whether it is 0 goes by how the places fall into steps and parts.) A row whose softmax is not a
// number is NaN in the dims that hold none, and stays as it is. Rare: only the parts of blocks that met some
// are looked through (one at a place that all see: 16 tokens over 32 x 8192 168 -> 449 us, 64 over 1 x 131072 165 -> 351,
// 4096 after 4096 3.5 ms). In the attention kernel this took registers from its loops (168 -> 185 to 203 us without any).
__device__ __forceinline__ void odd_tile(const TreeAttention& a, uint32_t* words, const Share& tile, int block) {
    const CachedTokens& c = a.c;
    const Entry& x = tile.x;
    const int h = tile.h, rt = tile.rt;
    constexpr int kWords = 4 * kMergeWaves;   // of 32 places, looked at together
    constexpr int kOddLoads = 4;              // (more of them would take registers from the joining)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int P = c.page_size, bsh = P % 16 == 0 ? 4 : 3, eb = a.elem;
    const int tok0 = rt * a.tile_tokens, tile_n = min(a.tile_tokens, x.n - tok0);
    const int row = blockIdx.x * kMergeRows + (tid >> 5), i = a.by_group.of(row), g = row - i * a.group, d4 = 4 * (tid & 31);
    if (static_cast<int>(blockIdx.x) * kMergeRows >= tile_n * a.group) return;
    const int tok = i < tile_n ? tok0 + i : INT_MAX;
    const int end = x.start + (a.tree ? x.n : tok0 + tile_n);
    const int32_t* table = c.table + static_cast<size_t>(x.row) * c.table_stride;
    int hi = 0;   // of the part that is looked through: places from here on are not its
    // Place t's row of V; null where there is none. (t may be past 2^31, hi is not.)
    auto v_row = [&](uint32_t t, float& scale) {
        scale = 1.0f;
        if (t >= static_cast<uint32_t>(hi)) return static_cast<const unsigned char*>(nullptr);
        const int n = a.by_page.of(static_cast<int>(t)), page = table[n], s = static_cast<int>(t) - n * P;
        if (page < 0 || page >= c.num_pages) return static_cast<const unsigned char*>(nullptr);
        const size_t at = (static_cast<size_t>(page) * c.hkv + h) * P + s;
        if (c.scales) scale = __builtin_bit_cast(float, static_cast<uint32_t>(c.scales[2 * (at >> bsh) + 1]) << 23);
        return static_cast<const unsigned char*>(c.v_cache) + at * (kHeadDim * eb);
    };
    auto value = [&](const unsigned char* p, int d, float scale) {
        return f16_bits_to_f32(eb == 2 ? reinterpret_cast<const uint16_t*>(p)[d] : fp8x2_to_f16x2<false>(p[d], scale) & 0xffffu);
    };
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    auto look = [&](uint32_t base) {
        __syncthreads();
#pragma unroll 1
        for (int w = wave; w < kWords; w += kMergeWaves) {
            uint32_t odd = 0;
#pragma unroll 1
            for (int j0 = 0; j0 < 32; j0 += 4 * kOddLoads) {   // 16 lanes a row
                const unsigned char* p[kOddLoads];
                float scale[kOddLoads];
                u32x4 v[kOddLoads];
#pragma unroll
                for (int j = 0; j < kOddLoads; ++j) p[j] = v_row(base + 32 * w + j0 + 4 * j + (lane >> 4), scale[j]);
#pragma unroll
                for (int j = 0; j < kOddLoads; ++j) {
                    v[j] = u32x4{0, 0, 0, 0};
                    if (p[j] && eb == 2) v[j] = reinterpret_cast<const u32x4*>(p[j])[lane & 15];
                    if (p[j] && eb == 1) {
                        const u32x2 y = reinterpret_cast<const u32x2*>(p[j])[lane & 15];
                        v[j][0] = y[0], v[j][1] = y[1];
                    }
                }
#pragma unroll
                for (int j = 0; j < kOddLoads; ++j) {
                    if (eb == 1)
                        v[j] = u32x4{fp8x2_to_f16x2<false>(v[j][0], scale[j]), fp8x2_to_f16x2<true>(v[j][0], scale[j]),
                                     fp8x2_to_f16x2<false>(v[j][1], scale[j]), fp8x2_to_f16x2<true>(v[j][1], scale[j])};
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) any |= (v[j][e] & 0x7c00u) == 0x7c00u || (v[j][e] & 0x7c000000u) == 0x7c000000u;
                    const uint64_t lanes = __builtin_amdgcn_ballot_w64(any);
#pragma unroll
                    for (int r = 0; r < 4; ++r) odd |= (lanes >> (16 * r) & 0xffff) != 0 ? 1u << (j0 + 4 * j + r) : 0u;
                }
            }
            if (lane == 0) words[w] = odd;
        }
        __syncthreads();
        for (int w = 0; w < kWords; ++w) {
            if (words[w] == 0) continue;
            for (uint32_t mine = words[w] & visible(a, x, tok, static_cast<int>(base + 32 * w) - x.start); mine != 0; mine &= mine - 1) {
                float scale;
                const unsigned char* p = v_row(base + 32 * w + __builtin_ctz(mine), scale);
                for (int e = 0; e < 4; ++e) {
                    const float y = value(p, d4 + e, scale);
                    if (!__builtin_isfinite(y)) sums[e] += y;
                }
            }
        }
    };
    // The tile's parts are its units in this block and the next ones.
    const long unit0 = tile.w - tile.u0;
    const int  parts = min(static_cast<int>(divide(unit0 + tile.units - 1, tile.per)) + 1, static_cast<int>(gridDim.y)) - block;
    for (int k = 0; k < parts; ++k) {
        const int32_t* d = a.desc + kDesc * (block + k);
        if ((load_uniform(d, 4) | load_uniform(d, 5)) == 0) continue;
        const long u0 = max((block + k) * tile.per - unit0, static_cast<long>(kItemUnits));
        const long u1 = min((block + k + 1) * tile.per - unit0, static_cast<long>(tile.units));
        const uint32_t lo = static_cast<uint32_t>(uniform((u0 - kItemUnits) * a.step));
        hi = max(static_cast<int>(uniform(min((u1 - kItemUnits) * a.step, static_cast<long>(end)))), 0);
        for (uint32_t at = lo; at < static_cast<uint32_t>(hi); at += 32 * kWords) look(at);
    }
    if (tok == INT_MAX) return;
    _Float16* const out = reinterpret_cast<_Float16*>(a.out) + (x.t0 + tok) * a.out_stride + (h * a.group + g) * kHeadDim + d4;
    bool nan = false;
    for (int e = 0; e < 4; ++e) nan |= sums[e] == 0.f && out[e] != out[e];
    if (__builtin_amdgcn_ballot_w64(nan) >> (tid & 32) & 0xffffffffu) return;
    for (int e = 0; e < 4; ++e)
        if (!(sums[e] == 0.f)) out[e] = static_cast<_Float16>(sums[e] * c.v_scale);
}

// The tile that begins in block x and goes on in the next ones. (At most one begins in a block and
// is not whole there, its last: slot 1 of the block holds it; slot 0 the block's part of one that
// began before.) A tile's rows go round the XCDs: with blocks x in a row of the grid, tiles that begin
// in every 32nd block were all joined on one of the eight (64 tokens over 1 x 131072: 22 us).
// And values that are not finite, in the tiles that begin in block x.
__global__ __launch_bounds__(64 * kMergeWaves, 6) void tree_merge_kernel(const int32_t* __restrict__ desc, const TreeAttention a) {
    const int row = blockIdx.x * kMergeRows + (threadIdx.x >> 5);
    const int block = blockIdx.y, blocks = gridDim.y;
    const int32_t* d = desc + kDesc * block;
    const int n = min(load_uniform(d, 0), blocks - block);
    uint32_t odd = load_uniform(d, 4) | load_uniform(d, 5);
    if (n > 1) {
        for (int k = 1 + static_cast<int>(threadIdx.x & 63); k < n; k += 64) odd |= d[kDesc * k + 4] | d[kDesc * k + 5];
        const int i = a.by_group.of(row), g = row - i * a.group;
        if (i < load_uniform(d, 2)) {
            const int t = load_uniform(d, 1) + i, head = load_uniform(d, 3) * a.group + g;
            if (n <= 2) merge_row<2>(a, n, block, row, t, head);
            else if (n <= 4) merge_row<4>(a, n, block, row, t, head);
            else merge_row<8>(a, n, block, row, t, head);
        }
    }
    if (__builtin_amdgcn_ballot_w64(odd != 0) == 0) return;
    __shared__ Schedule sch;
    __shared__ uint32_t words[4 * kMergeWaves];
    walk(a, sch, blocks, block, a.step, [&](const Share& s) {
        if (s.u0 <= kItemUnits) odd_tile(a, words, s, block);
    });
}

// Blocks on a CU. fp16: one of 8 waves; FP8, whose steps are half as many bytes: two of 4 waves
// up to 128 rows. us with two of 4 and with one of 8: fp16, 32 x 8192, 4 and 32 tokens 175 / 171 and
// 232 / 219, 37 ragged sequences, 8 tokens 45.5 / 41.6; FP8, 64 x 8192, 8 tokens 200 / 212, 37 ragged
// 36.4 / 38.1; block scales, 64 x 8192, 32 tokens 348 / 362.
constexpr bool small_blocks(int eb, int rows) { return eb == 1 && rows <= 128; }

template <int EB, bool BS, bool UNI, int ROWS>
void launch_r(TreeAttention& a, hipStream_t s) {
    constexpr int WQ = ROWS / 32, WK = (small_blocks(EB, ROWS) ? 4 : 8) / WQ;
    a.elem = EB;
    a.step = TreeKernel<EB, BS, WQ, WK, UNI>::kStep;
    hipLaunchKernelGGL((tree_attention_kernel<EB, BS, WQ, WK, UNI>), dim3(a.grid), dim3(64 * WQ * WK), 0, s, a);
}
template <int EB, bool BS, bool UNI>
void launch_u(TreeAttention& a, hipStream_t s) {
    switch (a.rows) {
        case 64: launch_r<EB, BS, UNI, 64>(a, s); break;
        case 128: launch_r<EB, BS, UNI, 128>(a, s); break;
        default: launch_r<EB, BS, UNI, 256>(a, s); break;
    }
}
template <int EB, bool BS>
void launch_e(TreeAttention& a, hipStream_t s) {
    if (a.c.page_size % 4 == 0) launch_u<EB, BS, true>(a, s);
    else if constexpr (!BS) launch_u<EB, false, false>(a, s);
}

int device_cus() {
    int dev = 0, n = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    hip_check(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev), "hipDeviceGetAttribute");
    return n;
}

}  // namespace

// Rows of a tile: those of an average entry, if no more than 256. us with 64, 128 and 256: fp16,
// 32 x 8192, 16 tokens of 4 heads a kv head (64 rows) 171 / 192 / 222, 32 tokens (128) 344 / 224 / 246;
// FP8, 1 x 131072, 64 tokens (256) 244 / 192 / 169; 4096 tokens after 4096 785 / 597 / 447. (Tiles of
// 32 rows, every wave a stream of its own, lost to 64: 4 tokens over 32 x 8192 197 / 170, 8 over
// 1 x 200 17.2 / 11.1; FP8 64 x 8192, 8 tokens, block scales 197 / 203.)
void tree_shape(int dtype, TreeAttention& a) {
    const long per = (static_cast<long>(a.c.n_tok) * a.group + a.c.n_ent - 1) / std::max(a.c.n_ent, 1);   // rows of an entry
    a.rows        = per <= 64 ? 64 : per <= 128 ? 128 : 256;
    a.tile_tokens = a.rows / a.group;
    a.by_tile     = place_div(a.tile_tokens);
    a.grid = device_cus() * (small_blocks(dtype == PA_KV_FP16 ? 2 : 1, a.rows) ? 2 : 1);
}

size_t tree_workspace(const TreeAttention& a) {
    return static_cast<size_t>(2 * a.grid) * a.rows * (kHeadDim + 2) * sizeof(float) +
           static_cast<size_t>(a.grid) * kDesc * sizeof(int32_t);
}

void tree_place(TreeAttention& a, void* workspace) {
    const size_t rows = static_cast<size_t>(2 * a.grid) * a.rows;
    a.part_out = static_cast<float*>(workspace);
    a.part_ml  = a.part_out + rows * kHeadDim;
    a.desc     = reinterpret_cast<int32_t*>(a.part_ml + 2 * rows);
}

hipError_t launch_tree_attention(int dtype, TreeAttention a, hipStream_t s) {
    check_kv_dtype(dtype);
    if (dtype == PA_KV_FP16) launch_e<2, false>(a, s);
    else if (dtype == PA_KV_FP8_E4M3) launch_e<1, false>(a, s);
    else launch_e<1, true>(a, s);
    hipLaunchKernelGGL(tree_merge_kernel, dim3(a.rows / kMergeRows, a.grid), dim3(64 * kMergeWaves), 0, s, a.desc, a);
    return hipGetLastError();
}

}  // namespace pa
