// fp4.h -- the 4-bit caches' numbers: E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives, the even channel in a byte's low half) and one power of two 2^e
// a 32 channels, held as the byte e + 127.
//
// e is the least with max|x| < 7 * 2^e: the largest value then rounds to 4 or 6
// times 2^e, and no value is off by more than half a step.  It is at least -23 and
// at most 13, so that every number of a cache is an FP16 number (half of 2^-23 is
// its least, 6 * 2^13 lies below its largest): attention multiplies FP16 operands
// that are exact.  The byte 255 stands for a block that is not finite.
#pragma once

#include "mixers.h"

namespace mqh {

constexpr int F4_BLOCK = 32;                    // channels of one scale
constexpr uint32_t F4_LOWEST = 127 - 23;        // the least scale byte
constexpr uint32_t F4_NONE = 255;               // a block that is not finite, or past what a scale reaches
constexpr uint32_t F4_FIRST_PAST = 0x47600000u; // the bits of 7 * 2^13

// a block's scale byte from the bits of its largest magnitude: a fraction of 1.75 or
// more carries into the exponent
__device__ __forceinline__ uint32_t f4_scale(uint32_t top) {
    if (top >= F4_FIRST_PAST) return F4_NONE;
    const int e = (int)((top + 0x200000u) >> 23) - 2;
    return (uint32_t)max(e, (int)F4_LOWEST);
}

__device__ __forceinline__ float f4_factor(uint32_t scale) { return __uint_as_float(scale << 23); }

// eight codes of one block as FP16 and as FP32 (each conversion takes two: a byte)
__device__ __forceinline__ uintx4 f4_to_half(uint32_t w, float factor) {
    return uintx4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 0)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 1)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 2)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 3))};
}
__device__ __forceinline__ void f4_to_float(uint32_t w, float factor, float (&x)[8]) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, factor, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, factor, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, factor, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, factor, 3);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
}
// eight values below 7 factors in size as codes, to nearest, ties to the even code
__device__ __forceinline__ uint32_t f4_codes(const float (&x)[8], float factor) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], factor, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], factor, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], factor, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], factor, 3);
}

}  // namespace mqh
