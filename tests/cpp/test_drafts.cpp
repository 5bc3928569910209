// The C++ surface of the drafted-token operators (decode/drafts.hpp).
//
//   test_drafts cpu   refusals that need no device
//   test_drafts gpu   a step of drafted tokens over a PagedKVCache's pages: appended, read
//                     back, attended (against attention in 64 bits over the rows read back),
//                     the accepted ones kept
//
// Exit status 0 = every check passed; each failure prints one line.

#include "decode/drafts.hpp"
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

template <class F>
void expect_refused(F&& f, const std::string& what) {
    try {
        f();
        expect(false, what + " (no exception)");
    } catch (const std::invalid_argument&) {
    } catch (const std::exception& e) {
        expect(false, what + " (wrong exception: " + e.what() + ")");
    }
}

constexpr int kD = 128;

void cpu_checks() {
    using namespace decode;
    const HeadRows q;
    pa_cached_tokens c{};
    expect_refused([&] { tree_attention(KVDtype::FP16, c, q, nullptr, 0, 1.0f, nullptr, 0); }, "attention: empty cache");
    expect_refused([&] { (void)tree_attention_workspace(KVDtype::FP16, c, 8); }, "workspace: empty cache");
    expect_refused([&] { keep_rows(KVDtype::FP16, c, nullptr, 1, nullptr); }, "keep_rows: empty cache");
    expect_refused([&] { read_cache(KVDtype::FP16, c, ValueType::FP32, nullptr, 0, nullptr, 0); }, "read_cache: empty cache");
    c.page_size = 12;
    c.num_kv_heads = c.block_table_stride = 1;
    expect_refused([&] { keep_rows(KVDtype::FP8_E4M3_BLOCK, c, nullptr, 0, nullptr); }, "block scales on pages of 12");
    keep_rows(KVDtype::FP8_E4M3, c, nullptr, 0, nullptr);   // nothing to do
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

void gpu_step(decode::KVDtype dtype) {
    using namespace decode;
    const int hq = 8, hkv = 2, P = 24, start = 50, m = 6, slots = 2;
    PagedKVCache::Config cfg{};
    cfg.num_pages = 12;
    cfg.page_size = P;
    cfg.num_kv_heads = hkv;
    cfg.head_dim = kD;
    cfg.max_slots = slots;
    cfg.max_pages_per_slot = 6;
    cfg.dtype = dtype;
    if (dtype == KVDtype::FP8_E4M3) cfg.k_scale = cfg.v_scale = 6.0f / 448.0f;
    PagedKVCache cache(cfg);
    std::mt19937 rng(11);
    std::normal_distribution<float> normal;
    const int n = slots * (start + m), row = (hq + 2 * hkv) * kD;
    std::vector<uint16_t> x(static_cast<size_t>(n) * row);
    for (uint16_t& e : x) e = orc_f32_to_f16(normal(rng));
    half* dx = reinterpret_cast<half*>(to_device(x));
    half* dout = nullptr;
    (void)hipMalloc(reinterpret_cast<void**>(&dout), static_cast<size_t>(slots) * m * hq * kD * 2);
    HeadRows k, q;
    k.in = dx + hq * kD;
    k.in_stride = q.in_stride = row;
    k.heads = hkv;
    expect(cache.admit() == 0 && cache.admit() == 1, "two slots");
    expect(cache.append_rope({0, 1}, {start, start}, nullptr, nullptr, k, dx + (hq + hkv) * kD, row), "prompts");
    k.in += static_cast<size_t>(slots) * start * row;
    expect(cache.append_rope({0, 1}, {m, m}, nullptr, nullptr, k, dx + static_cast<size_t>(slots) * start * row + (hq + hkv) * kD, row),
           "drafted tokens");

    const DecodeParams p = cache.params();
    int32_t *begin = to_device(std::vector<int32_t>{0, m, 2 * m}), *starts = to_device(std::vector<int32_t>{start, start});
    pa_cached_tokens c{};
    c.num_tokens = slots * m;
    c.num_entries = slots;
    c.tok_begin = begin;
    c.start_pos = starts;
    c.k_cache = const_cast<void*>(p.k_cache);
    c.v_cache = const_cast<void*>(p.v_cache);
    c.kv_scales = const_cast<uint8_t*>(p.kv_scales);
    c.block_table = p.block_table;
    c.block_table_stride = cfg.max_pages_per_slot;
    c.num_table_rows = slots;
    c.num_pages = cfg.num_pages;
    c.page_size = P;
    c.num_kv_heads = hkv;
    c.k_scale = cfg.k_scale;
    c.v_scale = cfg.v_scale;

    // Everything that the sequences hold, read back.
    const int all = slots * (start + m);
    pa_cached_tokens whole = c;
    int32_t *wbegin = to_device(std::vector<int32_t>{0, start + m, all}), *zeros = to_device(std::vector<int32_t>{0, 0});
    whole.num_tokens = all;
    whole.tok_begin = wbegin;
    whole.start_pos = zeros;
    float *dk = nullptr, *dv = nullptr;
    const size_t elems = static_cast<size_t>(all) * hkv * kD;
    (void)hipMalloc(reinterpret_cast<void**>(&dk), elems * 4);
    (void)hipMalloc(reinterpret_cast<void**>(&dv), elems * 4);
    read_cache(dtype, whole, ValueType::FP32, dk, hkv * kD, dv, hkv * kD);
    const auto K = to_host<float>(dk, elems), V = to_host<float>(dv, elems);
    const double step = dtype == KVDtype::FP16 ? 0.0 : std::ldexp(1.0, -4);
    double off = 0;
    for (int s = 0; s < slots; ++s)
        for (int t = 0; t < start + m; ++t)
            for (int e = 0; e < hkv * kD; ++e) {
                const size_t src = t < start ? static_cast<size_t>(s) * start + t : static_cast<size_t>(slots) * start + s * m + t - start;
                const double want = orc_f16_to_f32(x[src * row + hq * kD + e]);
                off = std::max(off, std::fabs(K[(static_cast<size_t>(s) * (start + m) + t) * hkv * kD + e] - want) - std::fabs(want) * step);
            }
    expect(off < 1e-4, "rows read back within half a step of what was appended");

    // A tree: two branches of three tokens each.
    const std::vector<uint64_t> bits = {1, 2, 5, 10, 21, 42};
    std::vector<uint64_t> both(bits);
    both.insert(both.end(), bits.begin(), bits.end());
    uint64_t* tree = to_device(both);
    q.in = dx + static_cast<size_t>(slots) * start * row;
    q.out = dout;
    q.out_stride = hq * kD;
    q.heads = hq;
    const size_t need = tree_attention_workspace(dtype, c, hq);
    void* ws = nullptr;
    (void)hipMalloc(&ws, need);
    expect_refused([&] { tree_attention(dtype, c, q, tree, 1, 0.1f, ws, need - 1); }, "a workspace one byte short");
    tree_attention(dtype, c, q, tree, 1, 0.1f, ws, need);
    const auto out = to_host<uint16_t>(dout, static_cast<size_t>(slots) * m * hq * kD);
    double err = 0;
    for (int s = 0; s < slots; ++s)
        for (int i = 0; i < m; ++i)
            for (int h = 0; h < hq; ++h) {
                std::vector<double> pr, o(kD);
                double den = 0;
                for (int t = 0; t < start + m; ++t) {
                    if (t >= start && !(bits[i] >> (t - start) & 1)) {
                        pr.push_back(0);
                        continue;
                    }
                    double dot = 0;
                    for (int d = 0; d < kD; ++d)
                        dot += static_cast<double>(orc_f16_to_f32(x[(static_cast<size_t>(slots) * start + s * m + i) * row + h * kD + d])) *
                               K[((static_cast<size_t>(s) * (start + m) + t) * hkv + h / (hq / hkv)) * kD + d];
                    pr.push_back(std::exp(0.1 * dot));
                    den += pr.back();
                }
                for (int t = 0; t < start + m; ++t)
                    for (int d = 0; d < kD; ++d)
                        o[d] += pr[t] / den * V[((static_cast<size_t>(s) * (start + m) + t) * hkv + h / (hq / hkv)) * kD + d];
                for (int d = 0; d < kD; ++d)
                    err = std::max(err, std::fabs(orc_f16_to_f32(out[(static_cast<size_t>(s * m + i) * hq + h) * kD + d]) - o[d]));
            }
    // Values below 6: probabilities and results rounded to fp16, 2^-11 each, and scores' own errors.
    expect(err < 6 * std::ldexp(1.0, -9), "attention over the rows read back");

    // The branch 0, 2, 4 of the first sequence and 1 of the second stay.
    int32_t *kept = to_device(std::vector<int32_t>{0, 2, 4, 1, 0, 0}), *counts = to_device(std::vector<int32_t>{3, 1});
    keep_rows(dtype, c, kept, 3, counts);
    read_cache(dtype, whole, ValueType::FP32, dk, hkv * kD, nullptr, 0);
    const auto now = to_host<float>(dk, elems);
    const int from[2][3] = {{0, 2, 4}, {1, -1, -1}};
    bool moved = true;
    for (int s = 0; s < slots; ++s)
        for (int j = 0; j < 3 && from[s][j] >= 0; ++j)
            for (int e = 0; e < hkv * kD; ++e) {
                const double was = K[(static_cast<size_t>(s) * (start + m) + start + from[s][j]) * hkv * kD + e];
                const double is = now[(static_cast<size_t>(s) * (start + m) + start + j) * hkv * kD + e];
                // (Block scales: rounded again to the block's scale, below 2 * 6 / 448 here.)
                moved = moved && std::fabs(is - was) <= (dtype == KVDtype::FP8_E4M3_BLOCK ? std::fabs(was) * std::ldexp(1.0, -4) + 1e-3 : 0.0);
            }
    expect(moved, "accepted rows lie behind the sequence");
    for (void* d : {static_cast<void*>(dx), static_cast<void*>(dout), static_cast<void*>(begin), static_cast<void*>(starts),
                    static_cast<void*>(wbegin), static_cast<void*>(zeros), static_cast<void*>(dk), static_cast<void*>(dv),
                    static_cast<void*>(tree), ws, static_cast<void*>(kept), static_cast<void*>(counts)})
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
