// C-ABI host layer, part 4: new tokens of a step (pa_rope.hip): the rotation
// handle, head norms with rotation, appends with rotation into caller-owned
// caches. (The paged cache's own append is in pa_kvcache.cpp.)

#include "pa_host.hpp"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>
#include <string>
#include <vector>

namespace {

using namespace pa::host;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// One pass indexes (token, head, 8-dim chunk) in 32 bits.
void check_count(const char* what, long long n, long long heads) {
    if (n * heads * (pa::kHeadDim / 8) > INT_MAX)
        throw std::length_error(std::string(what) + ": tokens * heads * 16 exceeds INT_MAX");
}

// Heads of one operand: a wave's resource over a token's heads, and in a block
// 15 strides and the heads, stay below 2^31 bytes.
constexpr int kMaxHeads = 1 << 19;

// Elements from one token to the next.
bool stride_ok(int64_t s) { return s >= 0 && s < (1 << 26) && s % 8 == 0; }

// n rows of some heads, `step` bytes apart.
struct Rows {
    int64_t base, step, bytes;
};
Rows rows_at(const uint16_t* p, long long stride, int heads) {
    return {static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)), 2 * stride, 2ll * heads * pa::kHeadDim};
}
int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }   // b > 0

// Whether any of a's n rows shares a byte with any of b's. (Columns of one buffer
// lie between each other and do not.) Rows of one stride: whether a row's distance
// from some row of the other, which moves by that stride, falls inside it; else
// row by row, which only rows of different strides that lie among each other need.
bool meet(const Rows& a, const Rows& b, int n) {
    const int64_t last = n - 1;
    if (a.base >= b.base + last * b.step + b.bytes || b.base >= a.base + last * a.step + a.bytes) return false;
    auto hits = [&](int64_t from, int64_t bytes, int64_t first, int64_t steps) {   // of b's rows first .. steps
        if (b.step == 0) return from < b.base + b.bytes && b.base < from + bytes;
        const int64_t lo = std::max(first, floor_div(from - b.base - b.bytes, b.step) + 1);
        return lo <= steps && b.base + lo * b.step < from + bytes;
    };
    if (a.step == b.step) return hits(a.base, a.bytes, -last, last);
    for (int64_t i = 0; i <= last; ++i)
        if (hits(a.base + i * a.step, a.bytes, 0, last)) return true;
    return false;
}

// r's output against other rows (none where p is null) that the call reads or writes.
bool meets_output(const pa::HeadRows& r, const uint16_t* p, long long stride, int heads, int n) {
    return n > 0 && r.heads > 0 && heads > 0 && p &&
           meet(rows_at(r.out, r.out_stride, r.heads), rows_at(p, stride, heads), n);
}

}  // namespace

namespace pa::host {

pa::RopeTable rope_table(const pa_rope* rope) {
    pa::RopeTable t{};
    t.scale = 1.0f;
    if (!rope) return t;
    int dev = 0;
    pa::hip_check(hipGetDevice(&dev), "hipGetDevice");
    if (dev != rope->device) throw std::invalid_argument("rope: made on another device than the current one");
    t.half_turns  = rope->half_turns;
    t.axes        = rope->axes;
    t.pairs       = rope->rot_dim / 2;
    t.num_axes    = rope->num_axes;
    t.interleaved = rope->interleaved;
    t.scale       = rope->scale;
    return t;
}

pa::HeadRows head_rows(const char* what, const pa_head_rows* r, int n, bool has_out) {
    pa::HeadRows h{};
    if (!r || r->heads == 0) return h;
    const std::string w = std::string(what) + ": ";
    if (r->heads < 0) throw std::invalid_argument(w + "negative head count");
    if (r->heads > kMaxHeads) throw std::length_error(w + "more than 2^19 heads");
    check_count(what, n, r->heads);
    if (n > 0) {
        if (!r->in) throw std::invalid_argument(w + "null rows");
        if (!aligned(r->in, 16) || !stride_ok(r->in_stride))
            throw std::invalid_argument(w + "rows must be 16-byte aligned, their stride a multiple of 8 elements below 2^26");
        if (r->weight && !aligned(r->weight, 16)) throw std::invalid_argument(w + "the norm weight must be 16-byte aligned");
        if (r->weight && r->eps != 0.0f && !(r->eps >= FLT_MIN))   // (v_rsq_f32 takes subnormals for 0)
            throw std::invalid_argument(w + "eps must be 0 or a positive normal number");
    }
    if (n > 0 && has_out) {
        if (!r->out) throw std::invalid_argument(w + "null output");
        if (!aligned(r->out, 16) || !stride_ok(r->out_stride))
            throw std::invalid_argument(w + "outputs must be 16-byte aligned, their stride a multiple of 8 elements below 2^26");
        if (n > 1 && r->out_stride < static_cast<long long>(r->heads) * pa::kHeadDim)
            throw std::invalid_argument(w + "output rows overlap");
        if (!(r->in == r->out && (n == 1 || r->in_stride == r->out_stride)) &&
            meet(rows_at(r->in, r->in_stride, r->heads), rows_at(r->out, r->out_stride, r->heads), n))
            throw std::invalid_argument(w + "the output overlaps the rows (it may only be the rows themselves)");
    }
    h.in         = r->in;
    h.in_stride  = static_cast<long>(r->in_stride);
    h.out        = r->out;
    h.out_stride = static_cast<long>(r->out_stride);
    h.weight     = r->weight;
    h.eps        = r->eps;
    h.heads      = r->heads;
    return h;
}

void check_page_bytes(const char* what, int dtype, int page_size, int kv_heads) {
    if (static_cast<long long>(page_size) * kv_heads * pa::kHeadDim * (dtype == PA_KV_FP16 ? 2 : 1) > INT_MAX)
        throw std::invalid_argument(std::string(what) + ": page_size * kv heads * row bytes must be below 2^31");
}

void check_v_rows(const char* what, const uint16_t* v, int64_t stride, int n) {
    if (n > 0 && !v) throw std::invalid_argument(std::string(what) + ": v is null");
    if (n > 0 && (!aligned(v, 16) || !stride_ok(stride)))
        throw std::invalid_argument(std::string(what) +
                                    ": v must be 16-byte aligned, its stride a multiple of 8 elements below 2^26");
}

float inverse_scale(const char* what, int dtype, float scale) {
    if (dtype != PA_KV_FP8_E4M3) return 1.0f;
    const float inv = 1.0f / scale;
    if (!std::isfinite(inv) || inv == 0.0f)
        throw std::invalid_argument(std::string(what) + ": k_scale and v_scale must have finite reciprocals");
    return inv;
}

void check_outputs(const char* what, const pa::HeadRows& q, const pa::HeadRows& k, bool k_out, const uint16_t* v,
                   int64_t v_stride, int n) {
    const char* met = meets_output(q, k.in, k.in_stride, k.heads, n)                              ? "q's output overlaps k"
                      : meets_output(q, v, v_stride, k.heads, n)                                  ? "q's output overlaps v"
                      : k_out && meets_output(q, k.out, k.out_stride, k.heads, n)                 ? "the outputs overlap"
                      : k_out && meets_output(k, q.in, q.in_stride, q.heads, n)                   ? "k's output overlaps q"
                                                                                                  : nullptr;
    if (met) throw std::invalid_argument(std::string(what) + ": " + met);
}

}  // namespace pa::host

using namespace pa::host;

extern "C" {

pa_status pa_rope_create(const double* freqs, const int32_t* axes, int rot_dim, int num_axes, int interleaved,
                         float scale, pa_rope** out) {
    return guarded([&] {
        if (!freqs || !out) throw std::invalid_argument("rope: freqs or out is null");
        if (rot_dim < 16 || rot_dim > pa::kHeadDim || rot_dim % 16 != 0)
            throw std::invalid_argument("rope: rot_dim must be a multiple of 16 from 16 to 128");
        if (num_axes < 1 || num_axes > 4) throw std::invalid_argument("rope: 1 to 4 axes");
        if (num_axes > 1 && !axes) throw std::invalid_argument("rope: several axes need each pair's axis");
        if (!std::isfinite(scale)) throw std::invalid_argument("rope: scale must be finite");
        const int pairs = rot_dim / 2;
        // Half turns per position, then the axes.
        std::vector<unsigned char> host(static_cast<size_t>(pairs) * (sizeof(double) + sizeof(int32_t)));
        for (int i = 0; i < pairs; ++i) {
            if (!std::isfinite(freqs[i])) throw std::invalid_argument("rope: freqs must be finite");
            const double  half = static_cast<double>(freqs[i] / 3.14159265358979323846264338327950288L);
            const int32_t axis = axes ? axes[i] : 0;
            if (axis < 0 || axis >= num_axes) throw std::invalid_argument("rope: a pair's axis is out of range");
            std::memcpy(&host[static_cast<size_t>(i) * sizeof(double)], &half, sizeof half);
            std::memcpy(&host[static_cast<size_t>(pairs) * sizeof(double) + static_cast<size_t>(i) * sizeof(int32_t)],
                        &axis, sizeof axis);
        }
        auto* r = new pa_rope;
        try {
            r->rot_dim     = rot_dim;
            r->num_axes    = num_axes;
            r->interleaved = interleaved != 0;
            r->scale       = scale;
            pa::hip_check(hipGetDevice(&r->device), "hipGetDevice");
            pa::hip_check(hipMalloc(reinterpret_cast<void**>(&r->half_turns), host.size()), "hipMalloc rope");
            pa::hip_check(hipMemcpy(r->half_turns, host.data(), host.size(), hipMemcpyHostToDevice), "hipMemcpy rope");
            r->axes = reinterpret_cast<int32_t*>(r->half_turns + pairs);
        } catch (...) {
            (void)hipFree(r->half_turns);
            delete r;
            throw;
        }
        *out = r;
    });
}

void pa_rope_destroy(pa_rope* rope) {
    if (!rope) return;
    (void)hipFree(rope->half_turns);
    delete rope;
}
int pa_rope_dim(const pa_rope* rope) { return rope ? rope->rot_dim : 0; }
int pa_rope_axes(const pa_rope* rope) { return rope ? rope->num_axes : 0; }

pa_status pa_norm_rope(const pa_rope* rope, const pa_head_rows* q, const pa_head_rows* k, const int32_t* positions,
                       int n, void* stream) {
    return guarded([&] {
        if (n < 0) throw std::invalid_argument("norm_rope: negative token count");
        pa::RopeAppend a{};
        a.q = head_rows("norm_rope q", q, n, true);
        a.k = head_rows("norm_rope k", k, n, true);
        check_outputs("norm_rope", a.q, a.k, true, nullptr, 0, n);
        if (rope && n > 0 && !positions) throw std::invalid_argument("norm_rope: a rotation needs positions");
        check_count("norm_rope", n, static_cast<long long>(a.q.heads) + a.k.heads + 8);
        if (n == 0 || a.q.heads + a.k.heads == 0) return;
        a.rope      = rope_table(rope);
        a.positions = positions;
        a.n_tok     = n;
        pa::hip_check(pa::launch_norm_rope(a, as_stream(stream)), "norm_rope kernel launch");
    });
}

int pa_block_tokens(int page_size) { return pa::block_tokens(page_size); }

pa_status pa_append_rope(int dtype, const pa_append_args* p, const pa_rope* rope, const pa_head_rows* q,
                         const pa_head_rows* k, void* stream) {
    return guarded([&] {
        check_dtype(dtype);
        if (!p || !k) throw std::invalid_argument("append_rope: args or k is null");
        if (p->num_tokens < 0 || p->num_entries < 0 || p->page_size <= 0 || p->block_table_stride <= 0 ||
            p->num_table_rows < 0 || p->num_pages < 0)
            throw std::invalid_argument("append_rope: bad sizes");
        if (k->heads <= 0) throw std::invalid_argument("append_rope: k needs heads");
        const bool block = dtype == PA_KV_FP8_E4M3_BLOCK;
        check_page_bytes("append_rope", dtype, p->page_size, k->heads);
        if (block && pa::block_tokens(p->page_size) == 0)
            throw std::invalid_argument("append_rope: block-scaled caches need a page_size that is a multiple of 8");
        const int n = p->num_tokens;
        pa::RopeAppend a{};
        a.q = head_rows("append_rope q", q, n, true);
        a.k = head_rows("append_rope k", k, n, false);
        check_v_rows("append_rope", p->v, p->v_stride, n);
        check_outputs("append_rope", a.q, a.k, false, p->v, p->v_stride, n);
        check_count("append_rope", n, static_cast<long long>(a.q.heads) + 2ll * k->heads + 12);
        check_count("append_rope", p->num_entries, 128);
        if (n == 0) return;
        if (p->num_entries == 0) throw std::invalid_argument("append_rope: tokens of no entry");
        if (!p->tok_begin || !p->start_pos || !p->block_table || !p->k_cache || !p->v_cache)
            throw std::invalid_argument("append_rope: null pointer");
        if (!aligned(p->k_cache, 16) || !aligned(p->v_cache, 16))
            throw std::invalid_argument("append_rope: caches must be 16-byte aligned");
        if (block && (!p->kv_scales || !aligned(p->kv_scales, 2)))
            throw std::invalid_argument("append_rope: a block-scaled cache needs kv_scales (2-byte aligned)");
        if (rope && rope->num_axes > 1 && !p->positions)
            throw std::invalid_argument("append_rope: a rotation over several axes needs positions");
        a.inv_k        = inverse_scale("append_rope", dtype, p->k_scale);
        a.inv_v        = inverse_scale("append_rope", dtype, p->v_scale);
        a.rope         = rope_table(rope);
        a.v            = p->v;
        a.v_stride     = static_cast<long>(p->v_stride);
        a.positions    = p->positions;
        a.n_tok        = n;
        a.n_ent        = p->num_entries;
        a.tok_begin    = p->tok_begin;
        a.start        = p->start_pos;
        a.slot_ids     = p->slot_ids;
        a.table        = p->block_table;
        a.table_stride = p->block_table_stride;
        a.table_rows   = p->num_table_rows;
        a.num_pages    = p->num_pages;
        a.k_cache      = p->k_cache;
        a.v_cache      = p->v_cache;
        a.scales       = p->kv_scales;
        a.page_size    = p->page_size;
        pa::hip_check(pa::launch_append_rope(dtype, a, nullptr, 0, as_stream(stream)), "append_rope kernel launch");
    });
}

}  // extern "C"
