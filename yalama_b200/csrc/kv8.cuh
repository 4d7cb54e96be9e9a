// The 8-bit K/V cache: number formats and device helpers.
//
// A cache holds codes [hkv][cap][128] and one FP32 scale per block of tokens and
// head [hkv][ceil(cap / block)], for keys and for values; value = code x scale.
// Scales are powers of two (0: nothing but zeros in the block), the smallest
// with max |x| <= code_max x scale. That costs E4M3 nothing (a floating code has
// the same relative step at every scale) and INT8 up to one bit, and it makes
// the arithmetic around a scale exact: x / scale has x's own mantissa, so a code
// takes one rounding, and a block whose scale grows when a larger token joins it
// is rescaled by shifting exponents: E4M3 codes change only where they become
// subnormal (below 2^-6 of a unit), INT8 codes take one rounding to the coarser
// step.
#pragma once
#include "ylm_common.cuh"

namespace ylm {

constexpr int KV8_E4M3 = 0;
constexpr int KV8_INT8 = 1;

// Smallest power of two s with amax <= code_max * s (448 = 1.75 * 2^8, 127 =
// 1.984375 * 2^6); 0 for amax = 0. amax is an FP16 magnitude, so s is normal.
template <int FMT> __device__ __forceinline__ float kv8_scale_of(float amax)
{
    if (!(amax > 0.f))
        return 0.f;
    const uint32_t bits = __float_as_uint(amax);
    const uint32_t over = (bits & 0x7FFFFFu) > (FMT == KV8_E4M3 ? 0x600000u : 0x7E0000u) ? 1u : 0u;
    return __uint_as_float(((bits >> 23) + over - (FMT == KV8_E4M3 ? 8u : 6u)) << 23);
}

// Two values (already divided by the scale) to two codes, lo in the low byte.
// Round to nearest even; INT8 has no NaN code and stores 0 for NaN.
template <int FMT> __device__ __forceinline__ uint32_t kv8_encode2(float lo, float hi)
{
    if constexpr (FMT == KV8_E4M3)
    {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
        return r;
    }
    else
        return (uint32_t)(__float2int_rn(lo) & 0xFF) | ((uint32_t)(__float2int_rn(hi) & 0xFF) << 8);
}

// Four codes to four FP16 numbers, exactly: codes 0 and 1 in lo, 2 and 3 in hi.
template <int FMT> __device__ __forceinline__ void kv8_decode4(uint32_t c, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == KV8_E4M3)
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(c));
    else
    {
        // biased byte u = code + 128 under the exponent of 1024: the half 1024 + u, less 1152
        const uint32_t u = c ^ 0x80808080u, h0 = __byte_perm(u, 0x64646464u, 0x4140), h1 = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
        const __half2 d0 = __hsub2(*reinterpret_cast<const __half2 *>(&h0), bias);
        const __half2 d1 = __hsub2(*reinterpret_cast<const __half2 *>(&h1), bias);
        lo = *reinterpret_cast<const uint32_t *>(&d0);
        hi = *reinterpret_cast<const uint32_t *>(&d1);
    }
}

// Four codes to the codes of code * ratio (ratio <= 1 where the scale grew).
template <int FMT> __device__ __forceinline__ uint32_t kv8_rescale4(uint32_t c, float ratio)
{
    uint32_t lo, hi;
    kv8_decode4<FMT>(c, lo, hi);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
    const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return kv8_encode2<FMT>(f.x * ratio, f.y * ratio) | kv8_encode2<FMT>(g.x * ratio, g.y * ratio) << 16;
}

} // namespace ylm
