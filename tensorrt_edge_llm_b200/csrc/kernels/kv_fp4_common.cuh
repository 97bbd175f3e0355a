// Four-bit cache pages.  A layer is uint8 [pages, 2, Hkv, P, 9 D / 16]; the slab of a page, of its keys or values and of one head holds the
// codes [P, D / 2] (E2M1, the even feature in the low nibble) and behind them the block scales [P, D / 16] (E4M3, one per 16 features).  A value is
// code * block scale * scales[0 keys, 1 values].  A code has two significant bits and a block scale four, so code * block scale is exact in fp16.
#pragma once

#include <cuda_fp8.h>

#include "tc5_common.cuh"

namespace telb {

__device__ __forceinline__ size_t fp4_slab_bytes(int page_size, int d) { return (size_t)page_size * (d / 2 + d / 16); }

// Two codes (low nibble first) as half2 bits, four times over a word.
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(w));
}
// Two E4M3 bytes as half2 bits (low byte first).
__device__ __forceinline__ uint32_t e4m3x2_to_half(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ float e4m3_to_float(uint8_t b) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3))); }

// Codes of two values: the nearest level, halves to the even code.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
    uint16_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u16.u8 %0, t;\n\t}" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// A value before it is rounded to the type of the 16-bit copies: fp16 stops at its largest number.
template <typename T>
__device__ __forceinline__ float fp4_bound(float v) {
    if constexpr (std::is_same<T, __half>::value)
        if (fabsf(v) > 65504.f && fabsf(v) < INFINITY) v = copysignf(65504.f, v);
    return v;
}
template <typename T>
__device__ __forceinline__ T fp4_round(float v) { return Cvt<T>::from_f(fp4_bound<T>(v)); }

}  // namespace telb
