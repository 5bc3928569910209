// C-ABI host layer, part 5: drafted tokens over a caller's paged cache (pa_tree.hip,
// pa_rows.hip): attention of several new tokens per sequence, rows read back, accepted
// rows kept.

#include "pa_host.hpp"

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <string>

namespace {

using namespace pa::host;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Sizes that the kernels index in 32 bits.
constexpr int kMaxKvHeads = 1 << 14;
constexpr int kMaxEntries = 1 << 20;
constexpr int kMaxKeepItems = 1 << 25;   // entries times kv heads

// Sizes of a call, checked (no pointer is looked at).
void check_sizes(const char* what, int dtype, const pa_cached_tokens* c) {
    check_dtype(dtype);
    const std::string w = std::string(what) + ": ";
    if (!c) throw std::invalid_argument(w + "the cache is null");
    if (c->num_tokens < 0 || c->num_entries < 0 || c->page_size <= 0 || c->block_table_stride <= 0 ||
        c->num_table_rows < 0 || c->num_pages < 0 || c->num_kv_heads <= 0)
        throw std::invalid_argument(w + "bad sizes");
    if (c->num_kv_heads > kMaxKvHeads) throw std::length_error(w + "more than 2^14 kv heads");
    if (c->num_entries > kMaxEntries) throw std::length_error(w + "more than 2^20 entries");
    check_page_bytes(what, dtype, c->page_size, c->num_kv_heads);
    if (dtype == PA_KV_FP8_E4M3_BLOCK && pa::block_tokens(c->page_size) == 0)
        throw std::invalid_argument(w + "block-scaled caches need a page_size that is a multiple of 8");
}

// The kernels' form of a call that has work to do.
pa::CachedTokens cached_tokens(const char* what, int dtype, const pa_cached_tokens* c, bool tokens) {
    const std::string w = std::string(what) + ": ";
    const bool block = dtype == PA_KV_FP8_E4M3_BLOCK;
    if (!c->start_pos || !c->block_table || !c->k_cache || !c->v_cache || (tokens && !c->tok_begin))
        throw std::invalid_argument(w + "null pointer");
    if (!aligned(c->k_cache, 16) || !aligned(c->v_cache, 16))
        throw std::invalid_argument(w + "caches must be 16-byte aligned");
    if (block && (!c->kv_scales || !aligned(c->kv_scales, 2)))
        throw std::invalid_argument(w + "a block-scaled cache needs kv_scales (2-byte aligned)");
    if (dtype != PA_KV_FP16 && (!std::isfinite(c->k_scale) || !std::isfinite(c->v_scale)))
        throw std::invalid_argument(w + "k_scale and v_scale must be finite");
    pa::CachedTokens t{};
    t.tok_begin    = c->tok_begin;
    t.start        = c->start_pos;
    t.slot_ids     = c->slot_ids;
    t.table        = c->block_table;
    t.k_cache      = c->k_cache;
    t.v_cache      = c->v_cache;
    t.scales       = block ? c->kv_scales : nullptr;
    t.n_tok        = c->num_tokens;
    t.n_ent        = c->num_entries;
    t.table_stride = c->block_table_stride;
    t.table_rows   = c->num_table_rows;
    t.num_pages    = c->num_pages;
    t.page_size    = c->page_size;
    t.hkv          = c->num_kv_heads;
    t.k_scale      = dtype == PA_KV_FP16 ? 1.0f : c->k_scale;
    t.v_scale      = dtype == PA_KV_FP16 ? 1.0f : c->v_scale;
    t.by_page      = pa::page_div(c->page_size);
    return t;
}

struct Bytes {
    const void* p;
    size_t      n;
};
// What a call over cached tokens reads of its cache, table and entries.
std::array<Bytes, 7> reads_of(int dtype, const pa::CachedTokens& c) {
    const size_t rows = static_cast<size_t>(c.num_pages) * c.hkv * c.page_size;   // of a pool
    const size_t pool = rows * pa::kHeadDim * (dtype == PA_KV_FP16 ? 2 : 1);
    const size_t scales = c.scales ? 2 * rows / pa::block_tokens(c.page_size) : 0, ents = 4 * static_cast<size_t>(c.n_ent);
    return {{{c.k_cache, pool}, {c.v_cache, pool}, {c.scales, scales},
             {c.table, std::min(static_cast<size_t>(c.table_rows) * c.table_stride, size_t{1} << 58) * 4},
             {c.tok_begin, ents + 4}, {c.start, ents}, {c.slot_ids, ents}}};
}
// Refuses output rows that lie in what the call reads: other tokens' results would change under it.
void check_apart(const char* what, int dtype, const pa::CachedTokens& c, const void* out, int64_t stride, int64_t row, int elem) {
    for (const Bytes& b : reads_of(dtype, c))
        if (rows_touch(out, stride, row, elem, c.n_tok, b.p, b.n))
            throw std::invalid_argument(std::string(what) + ": an output overlaps the cache or another operand");
}

// The launch of an attention over c with hq query heads, its sizes checked.
pa::TreeAttention tree_sizes(int dtype, const pa_cached_tokens* c, int hq) {
    check_sizes("tree_attention", dtype, c);
    if (hq <= 0 || hq % c->num_kv_heads != 0 || hq / c->num_kv_heads > 32)
        throw std::invalid_argument("tree_attention: the query heads must be 1 to 32 times the kv heads");
    if (static_cast<long long>(c->num_tokens) * hq > pa::kMaxTreeRows)
        throw std::length_error("tree_attention: tokens * heads * 16 exceeds INT_MAX");
    pa::TreeAttention a{};
    a.c.n_tok = c->num_tokens;
    a.c.n_ent = c->num_entries;
    a.c.hkv   = c->num_kv_heads;
    a.group   = hq / c->num_kv_heads;
    a.by_page = pa::place_div(c->page_size);
    a.by_group = pa::place_div(a.group);
    return a;
}

}  // namespace

extern "C" {

pa_status pa_tree_attention_workspace(int dtype, const pa_cached_tokens* c, int num_q_heads, size_t* bytes) {
    return guarded([&] {
        if (!bytes) throw std::invalid_argument("tree_attention: bytes is null");
        pa::TreeAttention a = tree_sizes(dtype, c, num_q_heads);
        *bytes = 0;
        if (c->num_tokens == 0 || c->num_entries == 0) return;
        pa::tree_shape(dtype, a);
        *bytes = pa::tree_workspace(a);
    });
}

pa_status pa_tree_attention(int dtype, const pa_cached_tokens* c, const pa_head_rows* q, const uint64_t* tree,
                            int tree_words, float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        if (!q) throw std::invalid_argument("tree_attention: q is null");
        pa::TreeAttention a = tree_sizes(dtype, c, q->heads);
        if (q->weight) throw std::invalid_argument("tree_attention: q takes no norm weight");
        const pa::HeadRows r = head_rows("tree_attention q", q, c->num_tokens, true);
        if (tree && (tree_words <= 0 || !aligned(tree, 8)))
            throw std::invalid_argument("tree_attention: tree rows need words (8-byte aligned)");
        if (!std::isfinite(sm_scale)) throw std::invalid_argument("tree_attention: sm_scale must be finite");
        if (c->num_tokens == 0) return;
        if (c->num_entries == 0) throw std::invalid_argument("tree_attention: tokens of no entry");
        a.c = cached_tokens("tree_attention", dtype, c, true);
        if (c->num_pages == 0) throw std::invalid_argument("tree_attention: a cache of no pages");
        a.score_scale = sm_scale * a.c.k_scale * 1.44269504088896340736f;
        if (!std::isfinite(a.score_scale)) throw std::invalid_argument("tree_attention: sm_scale * k_scale must be finite");
        const int64_t row = static_cast<int64_t>(q->heads) * pa::kHeadDim;
        const Bytes   bits{tree, tree ? 8 * static_cast<size_t>(c->num_tokens) * tree_words : 0};
        check_apart("tree_attention", dtype, a.c, r.out, r.out_stride, row, 2);
        if (rows_touch(r.out, r.out_stride, row, 2, c->num_tokens, bits.p, bits.n))
            throw std::invalid_argument("tree_attention: the output overlaps the tree");
        pa::tree_shape(dtype, a);
        const size_t need = pa::tree_workspace(a);
        if (workspace_bytes < need || !workspace || !aligned(workspace, 16))
            throw std::invalid_argument("tree_attention: the workspace must have " + std::to_string(need) +
                                        " bytes, 16-byte aligned");
        bool apart = !rows_touch(r.in, r.in_stride, row, 2, c->num_tokens, workspace, need) &&
                     !rows_touch(r.out, r.out_stride, row, 2, c->num_tokens, workspace, need);
        for (const Bytes& b : reads_of(dtype, a.c)) apart = apart && !rows_touch(workspace, 0, static_cast<int64_t>(need), 1, 1, b.p, b.n);
        if (!apart || rows_touch(workspace, 0, static_cast<int64_t>(need), 1, 1, bits.p, bits.n))
            throw std::invalid_argument("tree_attention: the workspace overlaps an operand");
        a.q           = r.in;
        a.q_stride    = r.in_stride;
        a.out         = r.out;
        a.out_stride  = r.out_stride;
        a.tree        = tree;
        a.words       = tree_words;
        pa::tree_place(a, workspace);
        pa::hip_check(pa::launch_tree_attention(dtype, a, as_stream(stream)), "tree_attention kernel launch");
    });
}

pa_status pa_read_cache(int dtype, const pa_cached_tokens* c, int type, void* k_out, int64_t k_stride, void* v_out,
                        int64_t v_stride, void* stream) {
    return guarded([&] {
        check_sizes("read_cache", dtype, c);
        if (type != PA_VALUE_FP16 && type != PA_VALUE_BF16 && type != PA_VALUE_FP32)
            throw std::invalid_argument("read_cache: unknown value type " + std::to_string(type));
        const int n = c->num_tokens;
        const long long row = static_cast<long long>(c->num_kv_heads) * pa::kHeadDim;
        if (n * row > static_cast<long long>(INT_MAX) * 8) throw std::length_error("read_cache: tokens * heads * 16 exceeds INT_MAX");
        struct Out { void* p; int64_t stride; };
        for (const Out& o : {Out{k_out, k_stride}, Out{v_out, v_stride}}) {
            if (!o.p || n == 0) continue;
            if (!aligned(o.p, 16) || o.stride < 0 || o.stride >= (1 << 26) || o.stride % 8 != 0)
                throw std::invalid_argument(
                    "read_cache: outputs must be 16-byte aligned, their stride a multiple of 8 elements below 2^26");
            if (n > 1 && o.stride < row) throw std::invalid_argument("read_cache: output rows overlap");
        }
        if (n > 0 && k_out && v_out && rows_overlap(k_out, k_stride, v_out, v_stride, row, type == PA_VALUE_FP32 ? 4 : 2, n))
            throw std::invalid_argument("read_cache: the outputs overlap");
        if (n == 0 || (!k_out && !v_out)) return;
        if (c->num_entries == 0) throw std::invalid_argument("read_cache: tokens of no entry");
        pa::ReadCache a{};
        a.c        = cached_tokens("read_cache", dtype, c, true);
        for (const Out& o : {Out{k_out, k_stride}, Out{v_out, v_stride}})
            if (o.p) check_apart("read_cache", dtype, a.c, o.p, o.stride, row, type == PA_VALUE_FP32 ? 4 : 2);
        a.k_out    = k_out;
        a.k_stride = static_cast<long>(k_stride);
        a.v_out    = v_out;
        a.v_stride = static_cast<long>(v_stride);
        pa::hip_check(pa::launch_read_cache(dtype, type, a, as_stream(stream)), "read_cache kernel launch");
    });
}

pa_status pa_keep_rows(int dtype, const pa_cached_tokens* c, const int32_t* kept, int width, const int32_t* counts,
                       void* stream) {
    return guarded([&] {
        check_sizes("keep_rows", dtype, c);
        if (width < 0) throw std::invalid_argument("keep_rows: negative width");
        if (c->num_entries == 0 || width == 0) return;
        // (Block-scaled caches: 2^25 items would be 2^32 threads, one more than a launch holds.)
        const int most = std::min<long long>(kMaxKeepItems, UINT32_MAX / pa::keep_threads(dtype));
        if (static_cast<long long>(c->num_entries) * c->num_kv_heads > most)
            throw std::length_error("keep_rows: entries * kv heads exceeds " + std::string(most < kMaxKeepItems ? "2^25 - 1" : "2^25"));
        if (!kept || !counts) throw std::invalid_argument("keep_rows: null pointer");
        pa::KeepRows a{};
        a.c      = cached_tokens("keep_rows", dtype, c, false);
        a.kept   = kept;
        a.width  = width;
        a.counts = counts;
        pa::hip_check(pa::launch_keep_rows(dtype, a, as_stream(stream)), "keep_rows kernel launch");
    });
}

}  // extern "C"
