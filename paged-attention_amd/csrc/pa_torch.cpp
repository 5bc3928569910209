// Compiled torch binding of the decode path: class Decoder with the signature
// of the reference's bindings/torch_decode.cu:14-81 (plan(seq_lens, num_ctas),
// run(q, k_cache, v_cache, block_table, seq_lens_dev, k_scale, v_scale),
// num_ctas, num_segments), over the C ABI of libpa_decode.so. It runs on the
// current torch stream. Argument errors raise RuntimeError (TORCH_CHECK), the
// library's invalid-argument / length errors ValueError (pybind11's mapping of
// std::invalid_argument / std::length_error, as the reference's make_plan
// throws them), device errors RuntimeError.
//
// plan() builds the launch parameters that stay fixed between calls (shapes,
// softmax scale, the bound device plan); run() checks its tensors, allocates
// the output and fills in the per-call pointers and scales, then launches.

#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "pa_decode.h"

namespace {

void check_status(pa_status s) {
    if (s == PA_OK) return;
    const std::string msg = pa_last_error();
    if (s == PA_ERR_INVALID_ARGUMENT) throw std::invalid_argument(msg);
    if (s == PA_ERR_LENGTH) throw std::length_error(msg);
    throw std::runtime_error("paged decode: " + msg);
}

// [pages, num_kv_heads, blocks of a page, 2] scale bytes of a block-scaled cache.
void check_kv_scales(const torch::Tensor& s, const torch::Tensor& cache) {
    const int b = pa_block_tokens(static_cast<int>(cache.size(2)));
    TORCH_CHECK(b != 0, "block-scaled caches need a page_size that is a multiple of 8");
    TORCH_CHECK(s.is_cuda() && s.get_device() == cache.get_device() && s.is_contiguous() && s.element_size() == 1 &&
                    s.dim() == 4 && s.size(0) == cache.size(0) && s.size(1) == cache.size(1) &&
                    s.size(2) == cache.size(2) / b && s.size(3) == 2,
                "kv_scales must be a contiguous CUDA uint8 [pages, num_kv_heads, page_size / ", b,
                ", 2] tensor on the cache's device");
}

class Decoder {
public:
    Decoder(int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size, bool fp8,
            bool block_scales)
        : hq_(static_cast<int>(num_q_heads)),
          hkv_(static_cast<int>(num_kv_heads)),
          dim_(static_cast<int>(head_dim)),
          page_(static_cast<int>(page_size)),
          dtype_(block_scales ? PA_KV_FP8_E4M3_BLOCK : fp8 ? PA_KV_FP8_E4M3 : PA_KV_FP16) {
        TORCH_CHECK(fp8 || !block_scales, "block_scales needs fp8");
        TORCH_CHECK(!block_scales || pa_block_tokens(page_), "block_scales needs a page_size that is a multiple of 8");
        check_status(pa_device_plan_create(&dplan_));
    }
    ~Decoder() {
        pa_plan_destroy(plan_);
        pa_device_plan_destroy(dplan_);
    }
    Decoder(const Decoder&)            = delete;
    Decoder& operator=(const Decoder&) = delete;

    // torch_decode.cu:21-27: seq_lens is a CPU int32 tensor [batch].
    void plan(const torch::Tensor& seq_lens, int64_t num_ctas) {
        TORCH_CHECK(seq_lens.device().is_cpu() && seq_lens.scalar_type() == torch::kInt32,
                    "seq_lens must be a CPU int32 tensor");
        const torch::Tensor lens = seq_lens.contiguous();
        const int batch = static_cast<int>(lens.numel());
        pa_plan* next = nullptr;
        check_status(pa_plan_build(dtype_, lens.data_ptr<int32_t>(), batch, hq_, hkv_, dim_,
                                   static_cast<int>(num_ctas), &next));
        pa_plan_destroy(plan_);
        plan_ = next;
        const int device = c10::hip::current_device();
        check_status(pa_device_plan_upload(dplan_, plan_, hkv_ > 0 ? hq_ / hkv_ : 0, dim_,
                                           c10::hip::getCurrentHIPStream(device).stream()));
        int max_len = 0;
        const int32_t* l = lens.data_ptr<int32_t>();
        for (int i = 0; i < batch; ++i) max_len = std::max(max_len, l[i]);
        table_cols_ = (max_len + page_ - 1) / page_;
        batch_      = batch;
        tmpl_       = pa_decode_params{};
        tmpl_.batch        = batch;
        tmpl_.num_q_heads  = hq_;
        tmpl_.num_kv_heads = hkv_;
        tmpl_.head_dim     = dim_;
        tmpl_.page_size    = page_;
        tmpl_.sm_scale     = 1.0f / std::sqrt(static_cast<float>(dim_));
        check_status(pa_device_plan_bind(dplan_, &tmpl_));
    }

    // torch_decode.cu:31-59. q [batch, Hq, D] fp16; caches [pages, Hkv, P, D]
    // fp16 or one-byte FP8; block_table [batch, >= ceil(max len / P)] int32.
    torch::Tensor run(const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                      const torch::Tensor& block_table, const torch::Tensor& seq_lens_dev, double k_scale,
                      double v_scale, const std::optional<torch::Tensor>& kv_scales) {
        TORCH_CHECK(kv_scales.has_value() == (dtype_ == PA_KV_FP8_E4M3_BLOCK),
                    "kv_scales goes with a Decoder of block_scales");
        TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kHalf && q.is_contiguous(),
                    "q must be a contiguous CUDA fp16 tensor");
        TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous() && block_table.is_contiguous(),
                    "caches and block_table must be contiguous");
        TORCH_CHECK(plan_ != nullptr && q.size(0) == batch_, "q batch does not match the plan");
        TORCH_CHECK(block_table.scalar_type() == torch::kInt32, "block_table must be int32");
        // Shape checks beyond the reference's: a mismatch would otherwise
        // become out-of-range device reads.
        TORCH_CHECK(q.dim() == 3 && q.size(1) == hq_ && q.size(2) == dim_, "q must be [batch, num_q_heads, head_dim]");
        const int64_t elem = dtype_ == PA_KV_FP16 ? 2 : 1;
        for (const torch::Tensor* c : {&k_cache, &v_cache})
            TORCH_CHECK(c->is_cuda() && c->dim() == 4 && c->size(1) == hkv_ && c->size(2) == page_ &&
                            c->size(3) == dim_ && c->element_size() == elem,
                        "k_cache / v_cache must be CUDA [pages, num_kv_heads, page_size, head_dim] tensors of ",
                        elem == 2 ? "fp16" : "one-byte FP8", " elements");
        TORCH_CHECK(block_table.is_cuda() && block_table.dim() == 2 && block_table.size(0) >= batch_ &&
                        block_table.size(1) >= table_cols_,
                    "block_table must be a CUDA [batch, >= ceil(max seq_len / page_size)] tensor");
        TORCH_CHECK(seq_lens_dev.is_cuda() && seq_lens_dev.scalar_type() == torch::kInt32,
                    "seq_lens must be a CUDA int32 tensor");
        if (kv_scales) check_kv_scales(*kv_scales, k_cache);
        torch::Tensor out = torch::empty_like(q);
        pa_decode_params p = tmpl_;
        p.kv_scales = kv_scales ? static_cast<const uint8_t*>(kv_scales->data_ptr()) : nullptr;
        p.q                  = static_cast<const uint16_t*>(q.data_ptr());
        p.out                = static_cast<uint16_t*>(out.data_ptr());
        p.k_cache            = k_cache.data_ptr();
        p.v_cache            = v_cache.data_ptr();
        p.block_table        = block_table.data_ptr<int32_t>();
        p.seq_lens           = seq_lens_dev.data_ptr<int32_t>();
        p.block_table_stride = static_cast<int32_t>(block_table.size(1));
        p.k_scale            = static_cast<float>(k_scale);
        p.v_scale            = static_cast<float>(v_scale);
        check_status(pa_decode(dtype_, &p, c10::hip::getCurrentHIPStream(q.get_device()).stream()));
        return out;
    }

    int64_t num_ctas() const { return pa_plan_num_ctas(plan_); }
    int64_t num_segments() const { return pa_plan_num_segments(plan_); }

private:
    int             hq_, hkv_, dim_, page_;
    int             dtype_;
    int             batch_      = 0;
    int             table_cols_ = 0;
    pa_plan*        plan_       = nullptr;
    pa_device_plan* dplan_      = nullptr;
    pa_decode_params tmpl_{};
};

using OptTensor = std::optional<torch::Tensor>;

// The tensors' device as the current one for a call.
struct OnDevice {
    int before = c10::hip::current_device();
    explicit OnDevice(int device) {
        if (device != before) c10::hip::set_device(static_cast<c10::DeviceIndex>(device));
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) c10::hip::set_device(static_cast<c10::DeviceIndex>(before));
    }
};

bool heads_ok(const torch::Tensor& x, int64_t n) {
    return x.is_cuda() && x.scalar_type() == torch::kHalf && x.dim() == 3 && x.size(0) == n && x.size(1) > 0 &&
           x.size(2) == 128 && x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) == 128);
}
int64_t row_stride(const torch::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1) * 128; }
uint16_t* u16(const torch::Tensor& x) { return static_cast<uint16_t*>(x.data_ptr()); }

// q or k [n, heads, 128], with its output (made here where none is given).
pa_head_rows rows_of(const char* name, const torch::Tensor& x, const OptTensor& weight, double eps, OptTensor* out,
                     int64_t n, int device) {
    TORCH_CHECK(heads_ok(x, n) && x.get_device() == device, name,
                " must be a CUDA fp16 [tokens, heads, 128] tensor whose heads are contiguous");
    pa_head_rows r{};
    r.in        = u16(x);
    r.in_stride = row_stride(x);
    r.heads     = static_cast<int32_t>(x.size(1));
    r.eps       = static_cast<float>(eps);
    if (weight) {
        TORCH_CHECK(weight->is_cuda() && weight->get_device() == device && weight->scalar_type() == torch::kFloat &&
                        weight->is_contiguous() && weight->numel() == 128,
                    name, "_weight must be a contiguous CUDA float32 tensor of 128");
        r.weight = static_cast<const float*>(weight->data_ptr());
    }
    if (out) {
        // (Past the dispatcher: half of torch::empty's 0.45 us, where a small call takes 5.)
        if (!out->has_value())
            *out = torch::Tensor(at::detail::empty_cuda({n, x.size(1), 128}, torch::kHalf, x.device(), std::nullopt));
        TORCH_CHECK(heads_ok(**out, n) && (*out)->get_device() == device && (*out)->size(1) == x.size(1), name,
                    "_out must be a CUDA fp16 tensor of the shape of ", name, " whose heads are contiguous");
        r.out        = u16(**out);
        r.out_stride = row_stride(**out);
    }
    return r;
}

const int32_t* positions_of(const OptTensor& positions, const pa_rope* rope, int64_t n, int device) {
    if (!positions) return nullptr;
    const int64_t axes = rope ? pa_rope_axes(rope) : positions->numel() / (n > 0 ? n : 1);
    TORCH_CHECK(positions->is_cuda() && positions->get_device() == device && positions->scalar_type() == torch::kInt32 &&
                    positions->is_contiguous() && positions->numel() == n * axes &&
                    (positions->dim() == 1 || (positions->dim() == 2 && positions->size(0) == n)),
                "positions must be a contiguous CUDA int32 [tokens] or [tokens, axes] tensor");
    return positions->data_ptr<int32_t>();
}

std::tuple<OptTensor, OptTensor> norm_rope(const OptTensor& q, const OptTensor& k, const OptTensor& positions,
                                           int64_t rope_handle, const OptTensor& q_weight, const OptTensor& k_weight,
                                           double eps, OptTensor q_out, OptTensor k_out) {
    TORCH_CHECK(q || k, "q or k is needed");
    const auto* rope = reinterpret_cast<const pa_rope*>(rope_handle);
    const torch::Tensor& any = q ? *q : *k;
    TORCH_CHECK(any.is_cuda() && any.dim() == 3, "q and k must be CUDA fp16 [tokens, heads, 128] tensors");
    const int64_t n = any.size(0);
    const int device = any.get_device();
    TORCH_CHECK(n <= INT_MAX, "too many tokens");
    pa_head_rows qr{}, kr{};
    if (q) qr = rows_of("q", *q, q_weight, eps, &q_out, n, device);
    if (k) kr = rows_of("k", *k, k_weight, eps, &k_out, n, device);
    const int32_t* pos = positions_of(positions, rope, n, device);
    const OnDevice on(device);
    check_status(pa_norm_rope(rope, q ? &qr : nullptr, k ? &kr : nullptr, pos, static_cast<int>(n),
                              c10::hip::getCurrentHIPStream(device).stream()));
    return {q ? q_out : OptTensor(), k ? k_out : OptTensor()};
}

OptTensor append_rope(const OptTensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_cache,
                      const torch::Tensor& v_cache, const torch::Tensor& block_table, const torch::Tensor& tok_begin,
                      const torch::Tensor& start_pos, int64_t rope_handle, const OptTensor& positions,
                      const OptTensor& q_weight, const OptTensor& k_weight, double eps, double k_scale, double v_scale,
                      const OptTensor& kv_scales, const OptTensor& slot_ids, OptTensor q_out) {
    const auto* rope = reinterpret_cast<const pa_rope*>(rope_handle);
    TORCH_CHECK(k.is_cuda() && k.dim() == 3, "k must be a CUDA fp16 [tokens, heads, 128] tensor");
    const int64_t n = k.size(0);
    const int device = k.get_device();
    TORCH_CHECK(n <= INT_MAX, "too many tokens");
    pa_head_rows qr{};
    if (q) qr = rows_of("q", *q, q_weight, eps, &q_out, n, device);
    const pa_head_rows kr = rows_of("k", k, k_weight, eps, nullptr, n, device);
    TORCH_CHECK(heads_ok(v, n) && v.get_device() == device && v.size(1) == k.size(1),
                "v must be a CUDA fp16 tensor of k's shape whose heads are contiguous");
    for (const torch::Tensor* c : {&k_cache, &v_cache})
        TORCH_CHECK(c->is_cuda() && c->get_device() == device && c->is_contiguous() && c->dim() == 4 &&
                        c->size(0) <= INT_MAX && c->size(1) == k.size(1) && c->size(2) > 0 && c->size(2) <= INT_MAX &&
                        c->size(3) == 128 && c->sizes() == k_cache.sizes() &&
                        (c->scalar_type() == torch::kHalf || c->element_size() == 1) &&
                        c->scalar_type() == k_cache.scalar_type(),
                    "k_cache and v_cache must be contiguous CUDA [pages, k's heads, page_size, 128] tensors, both fp16 "
                    "or both one-byte FP8");
    const bool fp16 = k_cache.scalar_type() == torch::kHalf;
    TORCH_CHECK(!kv_scales || !fp16, "kv_scales goes with one-byte FP8 caches");
    if (kv_scales) check_kv_scales(*kv_scales, k_cache);
    auto ints = [&](const torch::Tensor& t, int64_t size, const char* what) {
        TORCH_CHECK(t.is_cuda() && t.get_device() == device && t.scalar_type() == torch::kInt32 && t.is_contiguous() &&
                        t.dim() == 1 && (size < 0 || t.size(0) == size) && t.size(0) <= INT_MAX,
                    what);
        return t.data_ptr<int32_t>();
    };
    pa_append_args a{};
    a.num_tokens  = static_cast<int32_t>(n);
    a.start_pos   = ints(start_pos, -1, "start_pos must be a contiguous CUDA int32 [entries] tensor");
    const int64_t m = start_pos.size(0);
    a.num_entries = static_cast<int32_t>(m);
    a.tok_begin   = ints(tok_begin, m + 1, "tok_begin must be a contiguous CUDA int32 [entries + 1] tensor");
    if (slot_ids) a.slot_ids = ints(*slot_ids, m, "slot_ids must be a contiguous CUDA int32 [entries] tensor");
    TORCH_CHECK(block_table.is_cuda() && block_table.get_device() == device && block_table.scalar_type() == torch::kInt32 &&
                    block_table.is_contiguous() && block_table.dim() == 2 && block_table.size(1) > 0 &&
                    block_table.size(0) <= INT_MAX && block_table.size(1) <= INT_MAX,
                "block_table must be a contiguous CUDA int32 [rows, columns] tensor");
    a.positions          = positions_of(positions, rope, n, device);
    a.v                  = u16(v);
    a.v_stride           = row_stride(v);
    a.k_cache            = k_cache.data_ptr();
    a.v_cache            = v_cache.data_ptr();
    a.kv_scales          = kv_scales ? static_cast<uint8_t*>(kv_scales->data_ptr()) : nullptr;
    a.block_table        = block_table.data_ptr<int32_t>();
    a.block_table_stride = static_cast<int32_t>(block_table.size(1));
    a.num_table_rows     = static_cast<int32_t>(block_table.size(0));
    a.num_pages          = static_cast<int32_t>(k_cache.size(0));
    a.page_size          = static_cast<int32_t>(k_cache.size(2));
    a.k_scale            = static_cast<float>(k_scale);
    a.v_scale            = static_cast<float>(v_scale);
    const OnDevice on(device);
    check_status(pa_append_rope(kv_scales ? PA_KV_FP8_E4M3_BLOCK : fp16 ? PA_KV_FP16 : PA_KV_FP8_E4M3, &a, rope,
                                q ? &qr : nullptr, &kr, c10::hip::getCurrentHIPStream(device).stream()));
    return q ? q_out : OptTensor();
}

// Caches, table and places of a call over cached tokens (n of them; tok_begin null: none).
int cached_tokens_of(pa_cached_tokens& c, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                     const torch::Tensor& block_table, const torch::Tensor* tok_begin, const torch::Tensor& start_pos,
                     double k_scale, double v_scale, const OptTensor& kv_scales, const OptTensor& slot_ids, int64_t n) {
    const int device = k_cache.is_cuda() ? static_cast<int>(k_cache.get_device()) : -1;
    for (const torch::Tensor* x : {&k_cache, &v_cache})
        TORCH_CHECK(x->is_cuda() && x->get_device() == device && x->is_contiguous() && x->dim() == 4 &&
                        x->size(0) <= INT_MAX && x->size(1) > 0 && x->size(1) <= INT_MAX && x->size(2) > 0 &&
                        x->size(2) <= INT_MAX && x->size(3) == 128 && x->sizes() == k_cache.sizes() &&
                        (x->scalar_type() == torch::kHalf || x->element_size() == 1) &&
                        x->scalar_type() == k_cache.scalar_type(),
                    "k_cache and v_cache must be contiguous CUDA [pages, kv heads, page_size, 128] tensors, both fp16 "
                    "or both one-byte FP8");
    const bool fp16 = k_cache.scalar_type() == torch::kHalf;
    TORCH_CHECK(!kv_scales || !fp16, "kv_scales goes with one-byte FP8 caches");
    if (kv_scales) check_kv_scales(*kv_scales, k_cache);
    auto ints = [&](const torch::Tensor& t, int64_t size, const char* what) {
        TORCH_CHECK(t.is_cuda() && t.get_device() == device && t.scalar_type() == torch::kInt32 && t.is_contiguous() &&
                        t.dim() == 1 && (size < 0 || t.size(0) == size) && t.size(0) <= INT_MAX,
                    what);
        return t.data_ptr<int32_t>();
    };
    TORCH_CHECK(n >= 0 && n <= INT_MAX, "too many tokens");
    c.num_tokens = static_cast<int32_t>(n);
    c.start_pos  = ints(start_pos, -1, "start_pos must be a contiguous CUDA int32 [entries] tensor");
    const int64_t m = start_pos.size(0);
    c.num_entries = static_cast<int32_t>(m);
    if (tok_begin) c.tok_begin = ints(*tok_begin, m + 1, "tok_begin must be a contiguous CUDA int32 [entries + 1] tensor");
    if (slot_ids) c.slot_ids = ints(*slot_ids, m, "slot_ids must be a contiguous CUDA int32 [entries] tensor");
    TORCH_CHECK(block_table.is_cuda() && block_table.get_device() == device && block_table.scalar_type() == torch::kInt32 &&
                    block_table.is_contiguous() && block_table.dim() == 2 && block_table.size(1) > 0 &&
                    block_table.size(0) <= INT_MAX && block_table.size(1) <= INT_MAX,
                "block_table must be a contiguous CUDA int32 [rows, columns] tensor");
    c.k_cache            = k_cache.data_ptr();
    c.v_cache            = v_cache.data_ptr();
    c.kv_scales          = kv_scales ? static_cast<uint8_t*>(kv_scales->data_ptr()) : nullptr;
    c.block_table        = block_table.data_ptr<int32_t>();
    c.block_table_stride = static_cast<int32_t>(block_table.size(1));
    c.num_table_rows     = static_cast<int32_t>(block_table.size(0));
    c.num_pages          = static_cast<int32_t>(k_cache.size(0));
    c.page_size          = static_cast<int32_t>(k_cache.size(2));
    c.num_kv_heads       = static_cast<int32_t>(k_cache.size(1));
    c.k_scale            = static_cast<float>(k_scale);
    c.v_scale            = static_cast<float>(v_scale);
    return kv_scales ? PA_KV_FP8_E4M3_BLOCK : fp16 ? PA_KV_FP16 : PA_KV_FP8_E4M3;
}

torch::Tensor tree_attention(const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                             const torch::Tensor& block_table, const torch::Tensor& tok_begin,
                             const torch::Tensor& start_pos, const OptTensor& tree, double k_scale, double v_scale,
                             const OptTensor& kv_scales, const OptTensor& slot_ids, double sm_scale, OptTensor out) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, "q must be a CUDA fp16 [tokens, heads, 128] tensor");
    const int64_t n = q.size(0);
    const int device = q.get_device();
    pa_cached_tokens c{};
    const int dtype = cached_tokens_of(c, k_cache, v_cache, block_table, &tok_begin, start_pos, k_scale, v_scale,
                                       kv_scales, slot_ids, n);
    TORCH_CHECK(k_cache.get_device() == device, "q and the caches must be on one device");
    const pa_head_rows r = rows_of("q", q, OptTensor(), 0.0, &out, n, device);
    int words = 0;
    if (tree) {
        TORCH_CHECK(tree->is_cuda() && tree->get_device() == device && tree->scalar_type() == torch::kLong &&
                        tree->is_contiguous() && tree->dim() == 2 && tree->size(0) == n && tree->size(1) > 0 &&
                        tree->size(1) <= INT_MAX,
                    "tree must be a contiguous CUDA int64 [tokens, words] tensor");
        words = static_cast<int>(tree->size(1));
    }
    const OnDevice on(device);
    size_t bytes = 0;
    check_status(pa_tree_attention_workspace(dtype, &c, r.heads, &bytes));
    torch::Tensor ws;
    if (bytes) ws = torch::Tensor(at::detail::empty_cuda({static_cast<int64_t>(bytes)}, torch::kByte, q.device(), std::nullopt));
    check_status(pa_tree_attention(dtype, &c, &r, tree ? reinterpret_cast<const uint64_t*>(tree->data_ptr()) : nullptr,
                                   words, static_cast<float>(sm_scale), bytes ? ws.data_ptr() : nullptr, bytes,
                                   c10::hip::getCurrentHIPStream(device).stream()));
    return *out;
}

std::tuple<torch::Tensor, torch::Tensor> read_cache(const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                                    const torch::Tensor& block_table, const torch::Tensor& tok_begin,
                                                    const torch::Tensor& start_pos, int64_t n, int type,
                                                    double k_scale, double v_scale, const OptTensor& kv_scales,
                                                    const OptTensor& slot_ids, OptTensor k_out, OptTensor v_out) {
    pa_cached_tokens c{};
    const int dtype = cached_tokens_of(c, k_cache, v_cache, block_table, &tok_begin, start_pos, k_scale, v_scale,
                                       kv_scales, slot_ids, n);
    const int device = k_cache.get_device();
    const auto want = type == PA_VALUE_FP32 ? torch::kFloat : type == PA_VALUE_BF16 ? torch::kBFloat16 : torch::kHalf;
    for (OptTensor* o : {&k_out, &v_out}) {
        if (!o->has_value())
            *o = torch::Tensor(at::detail::empty_cuda({n, k_cache.size(1), 128}, want, k_cache.device(), std::nullopt));
        const torch::Tensor& x = **o;
        TORCH_CHECK(x.is_cuda() && x.get_device() == device && x.scalar_type() == want && x.dim() == 3 && x.size(0) == n &&
                        x.size(1) == k_cache.size(1) && x.size(2) == 128 && x.stride(2) == 1 &&
                        (x.size(1) == 1 || x.stride(1) == 128),
                    "k_out and v_out must be CUDA [tokens, kv heads, 128] tensors of the dtype asked for, their heads contiguous");
    }
    const OnDevice on(device);
    check_status(pa_read_cache(dtype, &c, type, k_out->data_ptr(), row_stride(*k_out), v_out->data_ptr(),
                               row_stride(*v_out), c10::hip::getCurrentHIPStream(device).stream()));
    return {*k_out, *v_out};
}

void keep_rows(const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& block_table,
               const torch::Tensor& kept, const torch::Tensor& counts, const torch::Tensor& start_pos,
               const OptTensor& kv_scales, const OptTensor& slot_ids) {
    pa_cached_tokens c{};
    const int dtype = cached_tokens_of(c, k_cache, v_cache, block_table, nullptr, start_pos, 1.0, 1.0, kv_scales,
                                       slot_ids, 0);
    const int device = k_cache.get_device();
    TORCH_CHECK(kept.is_cuda() && kept.get_device() == device && kept.scalar_type() == torch::kInt32 &&
                    kept.is_contiguous() && kept.dim() == 2 && kept.size(0) == c.num_entries && kept.size(1) <= INT_MAX,
                "kept must be a contiguous CUDA int32 [entries, width] tensor");
    TORCH_CHECK(counts.is_cuda() && counts.get_device() == device && counts.scalar_type() == torch::kInt32 &&
                    counts.is_contiguous() && counts.dim() == 1 && counts.size(0) == c.num_entries,
                "counts must be a contiguous CUDA int32 [entries] tensor");
    const OnDevice on(device);
    check_status(pa_keep_rows(dtype, &c, kept.data_ptr<int32_t>(), static_cast<int>(kept.size(1)),
                              counts.data_ptr<int32_t>(), c10::hip::getCurrentHIPStream(device).stream()));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Compiled torch binding of the MI355X paged decode path (libpa_decode.so)";
    pybind11::class_<Decoder>(m, "Decoder")
        .def(pybind11::init<int64_t, int64_t, int64_t, int64_t, bool, bool>(), pybind11::arg("num_q_heads"),
             pybind11::arg("num_kv_heads"), pybind11::arg("head_dim"), pybind11::arg("page_size"),
             pybind11::arg("fp8"), pybind11::arg("block_scales") = false)
        .def("plan", &Decoder::plan, pybind11::arg("seq_lens"), pybind11::arg("num_ctas") = 0)
        .def("run", &Decoder::run, pybind11::arg("q"), pybind11::arg("k_cache"), pybind11::arg("v_cache"),
             pybind11::arg("block_table"), pybind11::arg("seq_lens_dev"), pybind11::arg("k_scale"),
             pybind11::arg("v_scale"), pybind11::arg("kv_scales") = pybind11::none())
        .def_property_readonly("num_ctas", &Decoder::num_ctas)
        .def_property_readonly("num_segments", &Decoder::num_segments);
    // pa_amd.ops gives these their defaults and takes the rotation's handle.
    m.def("norm_rope", &norm_rope);
    m.def("append_rope", &append_rope);
    m.def("tree_attention", &tree_attention);
    m.def("read_cache", &read_cache);
    m.def("keep_rows", &keep_rows);
}
