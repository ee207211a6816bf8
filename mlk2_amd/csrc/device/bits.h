// Numbers in 8 and 4 bits as the operators hold them: a scale and codes.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace mlk {

/// Scale and the power of two that values and scale are taken times before
/// codes are taken from them: with a scale below 2^-100 their differences would
/// pass under the smallest f32. The products are exact.
struct Scale {
    float stored, s, up;   // s = stored * up
};

/// Of the largest magnitude's bits, as an unsigned number: above any finite
/// one's where a value was not finite.
__device__ __forceinline__ Scale scaleOf(uint32_t top, float largest) {
    Scale r;
    r.stored = top >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, top) / largest;
    r.up = r.stored < 0x1p-100f ? 0x1p100f : 1.0f;
    r.s = r.stored * r.up;
    return r;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

/// x / s rounded to the nearest whole number, half way to the even one, within
/// -127 .. 127; 0 for a scale of 0 or NaN. `inv` is 1 / s, rounded: the product is
/// off by one at most, and what x is past it, x - q s, is exact in one fma where
/// it is near half of s (x and q s are whole multiples of half a step of s).
__device__ __forceinline__ int codeI8(float x, const Scale& scale, float inv) {
    x *= scale.up;
    float q = rintf(x * inv);
    const float rest = __builtin_fmaf(-q, scale.s, x), half = 0.5f * scale.s, size = fabsf(rest);
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (size > half || (size == half && odd)) q += rest > 0.0f ? 1.0f : -1.0f;
    return scale.s > 0.0f ? static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f)) : 0;
}

/// The code of the 4-bit number nearest to x / s: the borders between
/// neighbours, times s, that |x| is past. A border half way takes the even code:
/// above it for the odd ones. An fma's sign is that of the exact difference.
__device__ __forceinline__ uint32_t codeFp4(float x, const Scale& scale) {
    const float y = fabsf(x) * scale.up, s = scale.s;
    uint32_t code = 0;
    if (s > 0.0f) {
        code += __builtin_fmaf(-0.25f, s, y) > 0.0f;
        code += __builtin_fmaf(-0.75f, s, y) >= 0.0f;
        code += __builtin_fmaf(-1.25f, s, y) > 0.0f;
        code += __builtin_fmaf(-1.75f, s, y) >= 0.0f;
        code += __builtin_fmaf(-2.5f, s, y) > 0.0f;
        code += __builtin_fmaf(-3.5f, s, y) >= 0.0f;
        code += __builtin_fmaf(-5.0f, s, y) > 0.0f;
    }
    return code | (__builtin_bit_cast(uint32_t, x) >> 31) << 3;
}

using F32x2 = float __attribute__((ext_vector_type(2)));

/// The numbers of byte I's two codes, the low half's first.
template <int I>
__device__ __forceinline__ F32x2 numbersOf(uint32_t word) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, I);
}

}  // namespace mlk
