// The C++ surface of the new-token operators (decode::Rope, norm_rope, append_rope,
// PagedKVCache::append_rope) and of the block-scaled cache.
//
//   test_new_tokens cpu   refusals that need no device
//   test_new_tokens gpu   a serving step through the cache: its values against the
//                         formulas in 64 bits, its output against attention over them
//
// Exit status 0 = every check passed; each failure prints one line.

#include "decode/paged_kv_cache.hpp"
#include "pa_oracle.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

namespace {

int g_failures = 0;

void expect(bool ok, const std::string& what) {
    if (!ok) {
        std::printf("FAIL: %s\n", what.c_str());
        ++g_failures;
    }
}

template <class E, class F>
void expect_throw(F&& f, const std::string& what) {
    try {
        f();
        expect(false, what + " (no exception)");
    } catch (const E&) {
    } catch (const std::exception& e) {
        expect(false, what + " (wrong exception: " + e.what() + ")");
    }
}

constexpr int kD = 128;

void cpu_checks() {
    using namespace decode;
    expect(std::string(kv_dtype_name(KVDtype::FP8_E4M3_BLOCK)) == pa_kv_dtype_name(PA_KV_FP8_E4M3_BLOCK), "dtype name");
    expect(kv_dtype_bytes(KVDtype::FP8_E4M3_BLOCK) == 1, "dtype bytes");
    expect_throw<std::invalid_argument>([] { Rope r(std::vector<double>(60, 1.0)); }, "rot_dim 120");
    expect_throw<std::invalid_argument>([] { Rope r(std::vector<double>(64, 1.0), {0, 1}); }, "axes of another length");
    expect_throw<std::invalid_argument>([] { Rope r(std::vector<double>(64, 1.0), {}, 3); }, "axes missing");
    HeadRows q;
    q.heads = 4;
    expect_throw<std::invalid_argument>([&] { norm_rope(nullptr, &q, nullptr, nullptr, 3); }, "null rows");
    expect_throw<std::invalid_argument>([&] { append_rope(KVDtype::FP16, pa_append_args{}, nullptr, nullptr, q); },
                                        "empty args");
    PagedKVCache::Config cfg{};
    cfg.num_pages = cfg.max_slots = cfg.max_pages_per_slot = 4;
    cfg.num_kv_heads = 2;
    cfg.head_dim = kD;
    cfg.page_size = 12;
    cfg.dtype = KVDtype::FP8_E4M3_BLOCK;
    expect_throw<std::invalid_argument>([&] { PagedKVCache c(cfg); }, "block scales on pages of 12");
    cfg.page_size = 16;
    cfg.v_scale = 2.0f;
    expect_throw<std::invalid_argument>([&] { PagedKVCache c(cfg); }, "block scales with a tensor scale");
}

template <class T>
T* to_device(const std::vector<T>& v) {
    T* d = nullptr;
    (void)hipMalloc(reinterpret_cast<void**>(&d), v.size() * sizeof(T));
    (void)hipMemcpy(d, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice);
    return d;
}
template <class T>
std::vector<T> to_host(const void* d, size_t n) {
    std::vector<T> v(n);
    (void)hipDeviceSynchronize();
    (void)hipMemcpy(v.data(), d, n * sizeof(T), hipMemcpyDeviceToHost);
    return v;
}

// A row normed and turned in 64 bits (half-split pairs over all 128 dims).
std::vector<double> turned(const uint16_t* x, const std::vector<float>& w, float eps, int pos,
                           const std::vector<double>& freqs) {
    std::vector<double> y(kD);
    double sq = 0;
    for (int d = 0; d < kD; ++d) {
        y[d] = orc_f16_to_f32(x[d]);
        sq += y[d] * y[d];
    }
    const double inv = 1 / std::sqrt(sq / kD + eps);
    for (int d = 0; d < kD; ++d) y[d] *= inv * w[d];
    for (int i = 0; i < kD / 2; ++i) {
        const double a = y[i], b = y[i + kD / 2], c = std::cos(pos * freqs[i]), s = std::sin(pos * freqs[i]);
        y[i] = a * c - b * s;
        y[i + kD / 2] = b * c + a * s;
    }
    return y;
}

void gpu_step(decode::KVDtype dtype) {
    using namespace decode;
    const int hq = 8, hkv = 2, P = 24, pages = 12;
    PagedKVCache::Config cfg{};
    cfg.num_pages = pages;
    cfg.page_size = P;
    cfg.num_kv_heads = hkv;
    cfg.head_dim = kD;
    cfg.max_slots = 3;
    cfg.max_pages_per_slot = 6;
    cfg.dtype = dtype;
    if (dtype == KVDtype::FP8_E4M3) cfg.k_scale = cfg.v_scale = 6.0f / 448.0f;
    PagedKVCache cache(cfg);
    std::vector<double> freqs(kD / 2);
    for (int i = 0; i < kD / 2; ++i) freqs[i] = std::pow(10000.0, -2.0 * i / kD);
    const Rope rope(freqs);
    std::mt19937 rng(7);
    std::normal_distribution<float> normal;
    std::vector<float> w(kD);
    for (float& x : w) x = 1.0f + 0.2f * normal(rng);
    float* dw = to_device(w);

    // One fused projection of 50 tokens: a prompt of 40 and one of 10.
    const int n = 50, row = (hq + 2 * hkv) * kD;
    std::vector<uint16_t> x(static_cast<size_t>(n) * row);
    for (uint16_t& e : x) e = orc_f32_to_f16(normal(rng));
    half* dx = reinterpret_cast<half*>(to_device(x));
    half* dq = nullptr;
    (void)hipMalloc(reinterpret_cast<void**>(&dq), static_cast<size_t>(n) * hq * kD * 2);
    HeadRows q, k;
    q.in = dx;
    q.in_stride = k.in_stride = row;
    q.out = dq;
    q.out_stride = hq * kD;
    q.weight = k.weight = dw;
    q.heads = hq;
    k.in = dx + hq * kD;
    k.heads = hkv;
    expect(cache.admit() == 0 && cache.admit() == 1, "two slots");
    expect(cache.append_rope({0, 1}, {40, 10}, &rope, &q, k, dx + (hq + hkv) * kD, row), "appended");
    expect(cache.seq_len(0) == 40 && cache.seq_len(1) == 10, "lengths");
    expect_throw<std::invalid_argument>([&] { cache.append_rope({0}, {1, 2}, &rope, nullptr, k, dx, row); }, "sizes");

    const auto gq = to_host<uint16_t>(dq, static_cast<size_t>(n) * hq * kD);
    double off = 0;
    for (int t = 0; t < n; ++t)
        for (int h = 0; h < hq; ++h) {
            const auto ref = turned(&x[static_cast<size_t>(t) * row + h * kD], w, q.eps, t < 40 ? t : t - 40, freqs);
            for (int d = 0; d < kD; ++d)
                off = std::max(off, std::fabs(orc_f16_to_f32(gq[(static_cast<size_t>(t) * hq + h) * kD + d]) - ref[d]) -
                                        std::fabs(ref[d]) * std::ldexp(1.0, -11));
        }
    expect(off < 1e-4, "q within half a step (and 32-bit arithmetic) of the formula");

    // What the cache holds, as values.
    const DecodeParams p = cache.params();
    const size_t eb = static_cast<size_t>(kv_dtype_bytes(dtype)), elems = static_cast<size_t>(pages) * hkv * P * kD;
    const auto kraw = to_host<uint8_t>(p.k_cache, elems * eb), vraw = to_host<uint8_t>(p.v_cache, elems * eb);
    std::vector<uint8_t> scales;
    if (dtype == KVDtype::FP8_E4M3_BLOCK) scales = to_host<uint8_t>(p.kv_scales, static_cast<size_t>(pages) * hkv * (P / 8) * 2);
    auto value = [&](const std::vector<uint8_t>& raw, int slot, int t, int h, int d, int kv) {
        const int page = cache.block_table(slot)[t / P];
        const size_t i = ((static_cast<size_t>(page) * hkv + h) * P + t % P) * kD + d;
        if (dtype == KVDtype::FP16) return static_cast<double>(orc_f16_to_f32(reinterpret_cast<const uint16_t*>(raw.data())[i]));
        const double code = orc_e4m3_to_f32(raw[i]);
        if (dtype == KVDtype::FP8_E4M3) return code * (6.0f / 448.0f);
        const uint8_t e = scales[2 * ((static_cast<size_t>(page) * hkv + h) * (P / 8) + t % P / 8) + kv];
        return code * std::ldexp(1.0, e - 127);
    };
    const double step = dtype == KVDtype::FP16 ? std::ldexp(1.0, -11) : std::ldexp(1.0, -4);
    double koff = 0, voff = 0;
    for (int t = 0; t < n; ++t)
        for (int h = 0; h < hkv; ++h) {
            const uint16_t* kr = &x[static_cast<size_t>(t) * row + (hq + h) * kD];
            const int slot = t < 40 ? 0 : 1, pos = t < 40 ? t : t - 40;
            const auto ref = turned(kr, w, k.eps, pos, freqs);
            for (int d = 0; d < kD; ++d) {
                const double v = orc_f16_to_f32(kr[hkv * kD + d]);
                koff = std::max(koff, std::fabs(value(kraw, slot, pos, h, d, 0) - ref[d]) - std::fabs(ref[d]) * step);
                voff = std::max(voff, std::fabs(value(vraw, slot, pos, h, d, 1) - v) - std::fabs(v) * step);
            }
        }
    expect(koff < 1e-4 && voff < 1e-4, "k and v within half a step of their type");

    // The last tokens' q attend.
    half *dlast = nullptr, *dout = nullptr;
    (void)hipMalloc(reinterpret_cast<void**>(&dlast), 2 * hq * kD * 2);
    (void)hipMalloc(reinterpret_cast<void**>(&dout), 2 * hq * kD * 2);
    (void)hipMemcpy(dlast, dq + static_cast<size_t>(39) * hq * kD, hq * kD * 2, hipMemcpyDeviceToDevice);
    (void)hipMemcpy(dlast + hq * kD, dq + static_cast<size_t>(49) * hq * kD, hq * kD * 2, hipMemcpyDeviceToDevice);
    cache.decode(dlast, dout, 2, hq);
    const auto out = to_host<uint16_t>(dout, 2 * hq * kD);
    double err = 0;
    for (int s = 0; s < 2; ++s)
        for (int h = 0; h < hq; ++h) {
            const int len = s ? 10 : 40;
            std::vector<float> qf(kD), K(static_cast<size_t>(len) * kD), V(K.size()), o(kD);
            for (int d = 0; d < kD; ++d) qf[d] = orc_f16_to_f32(gq[(static_cast<size_t>(s ? 49 : 39) * hq + h) * kD + d]);
            for (int t = 0; t < len; ++t)
                for (int d = 0; d < kD; ++d) {
                    K[static_cast<size_t>(t) * kD + d] = static_cast<float>(value(kraw, s, t, h / (hq / hkv), d, 0));
                    V[static_cast<size_t>(t) * kD + d] = static_cast<float>(value(vraw, s, t, h / (hq / hkv), d, 1));
                }
            orc_cpu_attention(qf.data(), K.data(), V.data(), o.data(), len, kD);
            for (int d = 0; d < kD; ++d)
                err = std::max(err, std::fabs(static_cast<double>(orc_f16_to_f32(out[(static_cast<size_t>(s) * hq + h) * kD + d])) - o[d]));
        }
    expect(err < 2e-3, "attention over what the cache holds");

    // The same rows through the stand-alone call: the same q.
    std::vector<int> pos(n);
    for (int t = 0; t < n; ++t) pos[t] = t < 40 ? t : t - 40;
    int* dpos = to_device(pos);
    (void)hipMemset(dq, 0, static_cast<size_t>(n) * hq * kD * 2);
    norm_rope(&rope, &q, nullptr, dpos, n);
    expect(to_host<uint16_t>(dq, gq.size()) == gq, "norm_rope and append_rope turn q alike");
    for (void* d : {static_cast<void*>(dw), static_cast<void*>(dx), static_cast<void*>(dq), static_cast<void*>(dlast),
                    static_cast<void*>(dout), static_cast<void*>(dpos)})
        (void)hipFree(d);
}

}  // namespace

int main(int argc, char** argv) {
    const std::string mode = argc > 1 ? argv[1] : "cpu";
    try {
        cpu_checks();
        if (mode == "gpu")
            for (const decode::KVDtype t : {decode::KVDtype::FP16, decode::KVDtype::FP8_E4M3, decode::KVDtype::FP8_E4M3_BLOCK})
                gpu_step(t);
    } catch (const std::exception& e) {
        std::printf("FAIL: unexpected exception: %s\n", e.what());
        ++g_failures;
    }
    std::printf("%s: %d failure(s)\n", mode.c_str(), g_failures);
    return g_failures == 0 ? 0 : 1;
}
