// Internal interface between the C-ABI host layer (pa_plan.cpp, pa_pool.cpp,
// pa_kvcache.cpp) and the gfx950 kernels (pa_decode.hip, pa_cache.hip). Not
// installed; callers use pa_decode.h.
#pragma once

#include "pa_decode.h"

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <stdexcept>
#include <string>

namespace pa {

// Raised by host code for a failed HIP runtime call; the C ABI maps it to
// PA_ERR_DEVICE.
struct DeviceError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void hip_check(hipError_t e, const char* what) {
    if (e != hipSuccess)
        throw DeviceError(std::string(what) + ": " + hipGetErrorName(e) + " (" + hipGetErrorString(e) + ")");
}

constexpr int kHeadDim     = 128;   // the only head_dim the path supports (decode.cu:31-38)
constexpr int kGroupTokens = 16;    // tokens per MFMA step of the decode kernel
#ifndef PA_BLOCK_UNITS
#define PA_BLOCK_UNITS 8
#endif
constexpr int kBlockUnits  = PA_BLOCK_UNITS;   // work units (waves) per block of the decode kernel
// 1: plans whose split (row, kv head) items span blocks are merged inside the
// split kernel (pa_decode_params.block_merge 2); 0: by the merge kernel.
#ifndef PA_CHAIN_MERGE
#define PA_CHAIN_MERGE 1
#endif

// Byte gap between the end of the K pool and the start of the V pool when both
// share one allocation. A wave reads the same (page, kv head) run of K and of
// V at once; pools at the same offset modulo a large power of two put those
// two reads on the same HBM banks, and on MI355X a decode step is then 3-7%
// slower (32 x 8192 fp16, 16-token pages: 163.2 against 158.4 us). 8 KiB was
// the best or near-best gap for fp16 and FP8 at page sizes 16 to 8192.
#ifndef PA_POOL_STAGGER
#define PA_POOL_STAGGER 8192
#endif
constexpr size_t kPoolStagger = PA_POOL_STAGGER;

inline void check_kv_dtype(int dtype) {
    if (dtype != PA_KV_FP16 && dtype != PA_KV_FP8_E4M3 && dtype != PA_KV_FP8_E4M3_BLOCK)
        throw std::invalid_argument("unknown kv dtype " + std::to_string(dtype));
}

// A merge is cut into tasks of 256 elements of an item's group x 128. A device
// plan holds one arrival counter per (task, item) (block_merge 2), then, on a
// 16-byte boundary, each item's first unit (block_merge 3): where those start,
// in int32 elements from the counters.
constexpr int    merge_tasks(int group) { return group > 2 ? group / 2 : 1; }
constexpr size_t plan_item_units(int items, int group) {
    return (static_cast<size_t>(merge_tasks(group)) * static_cast<size_t>(items) + 3) & ~size_t{3};
}

// Tokens per planning tile (decode.cu:43-45 tile_tokens). The gfx950 kernel
// consumes 16-token groups, so every 16-token boundary is a legal cut.
int kernel_tile_tokens(int dtype, int group);
// Decode work units (waves) resident per CU at the kernel's occupancy.
int kernel_units_per_cu(int dtype, int group);

// Throws std::invalid_argument for unsupported (dtype, head_dim, group);
// returns the launch status otherwise.
hipError_t launch_decode_split(int dtype, const pa_decode_params& p, hipStream_t s);
hipError_t launch_decode_merge(int dtype, const pa_decode_params& p, hipStream_t s);
hipError_t launch_append(int dtype, const uint16_t* k, const uint16_t* v, void* k_cache,
                         void* v_cache, const int32_t* bt_row, int start_pos, int n, int hkv,
                         int page_size, float inv_k, float inv_v, hipStream_t s);
// One launch of the batched append. meta (int32, device), for n_ent entries:
//   tok_begin[n_ent]  first token of each entry in k / v (prefix sums of the counts)
//   old_len[n_ent]    the slot's length before the entry
//   pl_begin[n_ent]   the entry's first page in pages[]
//   pages[n_pl]       per entry, the pages holding positions old_len .. old_len + count - 1
//   tab[2 n_tab]      new block-table entries: flat index, page
//   lens[2 n_len]     new lengths, one per distinct slot: slot, length
struct AppendBatch {
    const uint16_t* k;
    const uint16_t* v;
    void*           k_cache;
    void*           v_cache;
    const int32_t*  meta;
    int32_t*        table;
    int32_t*        seq_lens;
    int             n_ent, n_pl, n_tab, n_len, n_tok;
    int             hkv, page_size;
    float           inv_k, inv_v;
};
// `meta` (host, n_meta ints) goes over inside the kernel's arguments when it
// fits (append_meta_inline); else it is null and a.meta is on the device.
hipError_t launch_append_batch(int dtype, const AppendBatch& a, const int32_t* meta, size_t n_meta, hipStream_t s);
// Whether an append's meta of n ints fits the kernel arguments (4 KiB in all).
constexpr size_t kAppendInlineInts = 896;
constexpr bool   append_meta_inline(size_t n) { return n <= kAppendInlineInts; }
// tok / page_size and what is left, without a divide: a shift for powers of
// two (shift >= 0), else floor(tok * magic / 2^(31 + l)) with l = ceil(log2 P)
// and magic = floor(2^(31 + l) / P) + 1, stored as shift = ~(l - 1). Exact for
// 0 <= tok < 2^31: with r = tok mod P, tok * magic / 2^(31 + l) = tok / P + e and
// 0 < e <= tok / 2^(31 + l) < 2^-l <= 1 / P, so adding e to r / P <= (P - 1) / P stays below 1.
struct PageDiv {
    int      shift;
    uint32_t magic;
    __device__ __forceinline__ int page(int tok) const {
        return shift >= 0 ? tok >> shift : static_cast<int>(__umulhi(static_cast<uint32_t>(tok), magic) >> ~shift);
    }
};
inline PageDiv page_div(int page_size) {
    const uint32_t P = static_cast<uint32_t>(page_size);
    if ((P & (P - 1)) == 0) return {__builtin_ctz(P), 0u};
    const int l = 32 - __builtin_clz(P - 1);   // ceil(log2 P), at least 2
    return {~(l - 1), static_cast<uint32_t>((1ull << (31 + l)) / P + 1)};
}

// tok / d for 0 <= tok < 2^31 without a branch on d: floor(2 tok * magic / 2^(32 + l)), with l and
// magic as above (a power of two has l = log2 d and magic 2^31 + 1).
struct PlaceDiv {
    uint32_t magic;
    int      shift;
    __device__ __forceinline__ int of(int tok) const {
        return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(tok), magic) >> shift);
    }
};
inline PlaceDiv place_div(int d) {
    const int l = d <= 1 ? 0 : 32 - __builtin_clz(static_cast<uint32_t>(d) - 1);   // ceil(log2 d)
    return {static_cast<uint32_t>((1ull << (31 + l)) / static_cast<uint32_t>(d) + 1), l};
}

// Block-scaled caches: tokens per block, the exponents that a scale may have, and
// the largest code at the largest of them (240 * 2^8 = 61440; 448 * 2^8, and even
// 256 * 2^8, would be past fp16, which the decode kernel widens to).
constexpr int block_tokens(int page_size) { return page_size <= 0 || page_size % 8 ? 0 : page_size % 16 ? 8 : 16; }
constexpr int   kBlockExpMin = -32, kBlockExpMax = 8;
constexpr float kBlockTop    = 240.0f;

// A rotation on the device (pairs 0: none): half turns per position of each pair,
// and the axis whose position turns it.
struct RopeTable {
    const double*  half_turns;
    const int32_t* axes;
    int            pairs, num_axes, interleaved;
    float          scale;
};
// pa_head_rows, checked.
struct HeadRows {
    const uint16_t* in;
    long            in_stride;
    uint16_t*       out;
    long            out_stride;
    const float*    weight;
    float           eps;
    int             heads;
};
// One launch of head rows, with or without an append. Where the tokens go comes
// from the caller's device arrays (tok_begin, start, slot_ids, table), or is a
// cache's meta as for AppendBatch (meta, or the list kernels' arguments).
struct RopeAppend {
    RopeTable       rope;
    HeadRows        q, k;
    const uint16_t* v;
    long            v_stride;
    const int32_t*  positions;
    int             n_tok, n_ent;
    const int32_t*  tok_begin;
    const int32_t*  start;
    const int32_t*  slot_ids;
    const int32_t*  table;
    int             table_stride, table_rows, num_pages;
    const int32_t*  meta;
    int             n_pl, n_tab, n_len;
    int32_t*        new_table;
    int32_t*        new_lens;
    void*           k_cache;
    void*           v_cache;
    uint8_t*        scales;
    int             page_size;
    float           inv_k, inv_v;
    // Set by the launch: block-scaled caches' units (of 2^block_shift tokens), by_token
    // where a unit is a token; waves of a token, of its q, of its k; quotients by
    // these, and entries per token or unit.
    int             block_shift, units, by_token, head_groups;
    int             parts, parts_q, parts_k;
    PageDiv         by_page, by_parts;
    float           ent_rate;
};
template <int N>
struct RopeInline {
    RopeAppend a;
    alignas(16) int32_t meta[N];
};
// Ints of meta that fit the kernel arguments beside RopeAppend.
constexpr size_t kRopeInlineInts = 896;
static_assert(sizeof(RopeInline<kRopeInlineInts>) <= 4096, "kernel arguments are 4 KiB at most");
hipError_t launch_norm_rope(const RopeAppend& a, hipStream_t s);
hipError_t launch_append_rope(int dtype, const RopeAppend& a, const int32_t* meta, size_t n_meta, hipStream_t s);
// Tokens of several sequences in a paged cache (pa_cached_tokens, checked).
struct CachedTokens {
    const int32_t* tok_begin;
    const int32_t* start;
    const int32_t* slot_ids;
    const int32_t* table;
    void*          k_cache;
    void*          v_cache;
    uint8_t*       scales;
    int            n_tok, n_ent;
    int            table_stride, table_rows, num_pages, page_size, hkv;
    float          k_scale, v_scale;
    PageDiv        by_page;
};
// Tokens times query heads of an attention, at most (its rows are indexed in 32 bits, 8 dims at a time).
constexpr long kMaxTreeRows = INT_MAX / (kHeadDim / 8);
// Attention of those tokens over their sequences.
struct TreeAttention {
    CachedTokens    c;
    const uint16_t* q;
    long            q_stride;
    uint16_t*       out;
    long            out_stride;
    const uint64_t* tree;      // [n_tok][words], or null: a chain
    int             words;
    int             group;     // query heads of a kv head
    PlaceDiv        by_page, by_group;
    float           score_scale;   // of q k into base-2 exponents
    int             elem, step;    // set by the launch: bytes of a cached value, places of a step
    // Set by tree_shape, with the workspace.
    int             rows, tile_tokens, grid;
    PlaceDiv        by_tile;
    float*          part_out;  // [2 grid][rows][128]
    float*          part_ml;   // [2 grid][rows][2]
    int32_t*        desc;      // [grid][8], the tile that a block begins and others end, whether it met values that are not finite
};
// Chooses the launch from the call's sizes (host only, but for the device's CU count).
void   tree_shape(int dtype, TreeAttention& a);
size_t tree_workspace(const TreeAttention& a);
void   tree_place(TreeAttention& a, void* workspace);
hipError_t launch_tree_attention(int dtype, TreeAttention a, hipStream_t s);
// Rows of the caches into k_out / v_out (one may be null); out_type: pa_value_type.
struct ReadCache {
    CachedTokens c;
    void*        k_out;
    long         k_stride;
    void*        v_out;
    long         v_stride;
};
hipError_t launch_read_cache(int dtype, int out_type, const ReadCache& a, hipStream_t s);
// Accepted rows up in their sequences: kept [n_ent][width], counts [n_ent].
struct KeepRows {
    CachedTokens   c;
    const int32_t* kept;
    int            width;
    const int32_t* counts;
};
int        keep_threads(int dtype);   // of an entry and kv head
hipError_t launch_keep_rows(int dtype, const KeepRows& a, hipStream_t s);
// Stores one zero.
hipError_t launch_zero_int(int32_t* p, hipStream_t s);
// Copies n ints (rounded up to whole 16 bytes) from pinned host memory to the
// device with a kernel. Both ends are 16-byte aligned and have that room. Block i
// of stage_copy_blocks(n) stores `mark` at marks[i] (pinned host memory; null:
// none) once it has read its part.
constexpr size_t stage_copy_blocks(size_t n) { return (n + 1023) / 1024; }
hipError_t launch_stage_copy(const int32_t* host, int32_t* dev, size_t n, int32_t* marks, int32_t mark, hipStream_t s);
hipError_t launch_gather(int dtype, const void* cache, const int32_t* bt_row, int hkv,
                         int page_size, int kv_head, int len, void* out, hipStream_t s);
hipError_t launch_fill_bytes(void* buf, size_t bytes, int value, hipStream_t s);
// n elements fp32 -> fp16 (RNE) when to_half, else fp16 -> fp32.
hipError_t launch_convert(const void* in, void* out, size_t n, bool to_half, hipStream_t s);
hipError_t launch_stream_read_chunked(const void* buf, size_t bytes, int blocks, int threads, int unroll,
                                     uint32_t* sink, hipStream_t s);
hipError_t launch_stream_read(const void* buf, size_t bytes, int blocks, int threads, int unroll, bool nt,
                              uint32_t* sink, hipStream_t s);

}  // namespace pa
