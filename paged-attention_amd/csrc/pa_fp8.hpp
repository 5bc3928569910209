// FP8 E4M3 encoding shared by the kernels that write caches (pa_cache.hip,
// pa_rope.hip).
#pragma once

#include "pa_device.hpp"

namespace pa {

// FP8 E4M3 encoder, written from the OCP OFP8 definition (bias 7, max normal
// 448 = S.1111.110, NaN = S.1111.111, subnormals m * 2^-9): round to nearest
// even, finite overflow and infinities saturate to +-448, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3_encode(float x) {
    const uint32_t u    = __builtin_bit_cast(uint32_t, x);
    const uint32_t sign = (u >> 24) & 0x80u;
    const uint32_t a    = u & 0x7fffffffu;
    if (a > 0x7f800000u) return sign | 0x7fu;    // NaN
    if (a >= 0x43e00000u) return sign | 0x7eu;   // |x| >= 448: saturate
    if (a < 0x3c800000u) {                       // |x| < 2^-6: subnormal grid
        const float ax = __builtin_bit_cast(float, a);
        return sign | static_cast<uint32_t>(rintf(ax * 512.0f));   // 0..8; 8 is the min normal
    }
    const uint32_t man = a & 0x7fffffu;
    uint32_t q = (((a >> 23) - 120u) << 3) | (man >> 20);
    const uint32_t rem = man & 0xfffffu;
    if (rem > 0x80000u || (rem == 0x80000u && (q & 1u))) q += 1u;
    return sign | q;
}

__device__ __forceinline__ float f16_bits_to_f32(uint32_t h16) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h16)));
}

// E4M3 encode of eight values through gfx950's OCP FP8 conversion
// (v_cvt_scalef32_pk_fp8_f32, scale 1). Finite values are clamped to +-448
// beforehand (saturation, and infinities). The instruction writes every NaN as
// 0xff; a chunk holding a NaN has those bytes put right, which keep the sign
// (0x7f | sign), as the software path and the oracle do.
#ifndef PA_APPEND_HWCVT
#define PA_APPEND_HWCVT 1
#endif
constexpr bool kAppendHwCvt = PA_APPEND_HWCVT != 0;

typedef short v2i16 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float clamp_abs(float x, float top) { return __builtin_fminf(__builtin_fmaxf(x, -top), top); }

// `top`: the largest magnitude stored, 448 or less (an E4M3 value).
__device__ __forceinline__ u32x2 e4m3_encode8(float (&f)[8], float top = 448.0f) {
    u32x2 out = {0u, 0u};
    bool  nan = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) nan |= f[e] != f[e];
    if constexpr (!kAppendHwCvt) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            out[e >> 2] |= e4m3_encode(f[e] == f[e] ? clamp_abs(f[e], top) : f[e]) << (8 * (e & 3));
        return out;
    }
    uint32_t keep[2] = {0u, 0u}, nans[2] = {0u, 0u};   // bytes of NaNs, and what they hold
    if (__builtin_expect(nan, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (f[e] == f[e]) continue;
            keep[e >> 2] |= 0xffu << (8 * (e & 3));
            nans[e >> 2] |= (0x7fu | (__builtin_bit_cast(uint32_t, f[e]) >> 24 & 0x80u)) << (8 * (e & 3));
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = clamp_abs(f[e], top);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        v2i16 r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, f[4 * w + 0], f[4 * w + 1], 1.0f, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, f[4 * w + 2], f[4 * w + 3], 1.0f, true);
        out[w] = (__builtin_bit_cast(uint32_t, r) & ~keep[w]) | nans[w];
    }
    return out;
}

// E4M3 bytes of eight products float(x) * inv of fp16 x, each rounded to fp32
// first.
__device__ __forceinline__ u32x2 encode8(const u32x4 in, float inv) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f16_bits_to_f32((in[e >> 1] >> (16 * (e & 1))) & 0xffffu) * inv;
    return e4m3_encode8(f);
}

}  // namespace pa
