#pragma once
// New tokens of a step, over libpa_decode.so: head norms with rotation, and
// appends with rotation into paged caches (no counterparts in the reference).

#include "decode_types.hpp"
#include "hip_check.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <vector>

namespace decode {

// Some heads of every token (pa_head_rows): token t's head h starts at in + t *
// in_stride + h * 128. weight null: no norm. out where the call has an output.
struct HeadRows {
    const half*  in         = nullptr;
    int64_t      in_stride  = 0;
    half*        out        = nullptr;
    int64_t      out_stride = 0;
    const float* weight     = nullptr;
    float        eps        = 1e-6f;
    int          heads      = 0;
};

// A model's rotation on the current device (pa_rope): pair i turns by freqs[i]
// radians per position.
class Rope {
public:
    explicit Rope(const std::vector<double>& freqs, const std::vector<int>& axes = {}, int num_axes = 1,
                  bool interleaved = false, float scale = 1.0f) {
        if (!axes.empty() && axes.size() != freqs.size())
            throw std::invalid_argument("rope: freqs and axes differ in size");
        detail::check(pa_rope_create(freqs.data(), axes.empty() ? nullptr : axes.data(),
                                     2 * static_cast<int>(freqs.size()), num_axes, interleaved ? 1 : 0, scale, &h_));
    }
    ~Rope() { pa_rope_destroy(h_); }
    Rope(const Rope&)            = delete;
    Rope& operator=(const Rope&) = delete;
    const pa_rope* handle() const { return h_; }

private:
    pa_rope* h_ = nullptr;
};

namespace detail {
inline pa_head_rows abi(const HeadRows& r) {
    pa_head_rows a{};
    a.in         = reinterpret_cast<const uint16_t*>(r.in);
    a.in_stride  = r.in_stride;
    a.out        = reinterpret_cast<uint16_t*>(r.out);
    a.out_stride = r.out_stride;
    a.weight     = r.weight;
    a.eps        = r.eps;
    a.heads      = r.heads;
    return a;
}
}  // namespace detail

// q and k of n tokens normed and rotated into their outputs; positions (device)
// [n][axes], null only without a rotation.
inline void norm_rope(const Rope* rope, const HeadRows* q, const HeadRows* k, const int* positions, int n,
                      hipStream_t stream = 0) {
    const pa_head_rows qr = q ? detail::abi(*q) : pa_head_rows{}, kr = k ? detail::abi(*k) : pa_head_rows{};
    detail::check(pa_norm_rope(rope ? rope->handle() : nullptr, q ? &qr : nullptr, k ? &kr : nullptr, positions, n,
                               stream));
}

// Tokens of several sequences into caller-owned pages of any cache type
// (pa_append_args), k (and q) normed and rotated on the way.
inline void append_rope(KVDtype dtype, const pa_append_args& args, const Rope* rope, const HeadRows* q,
                        const HeadRows& k, hipStream_t stream = 0) {
    const pa_head_rows qr = q ? detail::abi(*q) : pa_head_rows{}, kr = detail::abi(k);
    detail::check(pa_append_rope(static_cast<int>(dtype), &args, rope ? rope->handle() : nullptr, q ? &qr : nullptr,
                                 &kr, stream));
}

}  // namespace decode
