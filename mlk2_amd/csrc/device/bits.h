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

/// codeI8 of E numbers, four to a word. x * inv, rounded once, lies within 2^-16 of
/// x / s, so it rounds to the same whole number unless it is that near to half way
/// between two: those are looked at as codeI8 does. Adding 1.5 * 2^23 leaves the
/// number in the low bits.
template <int E>
__device__ __forceinline__ void codesI8(const float (&x)[E], const Scale& scale, uint32_t (&words)[E / 4]) {
    constexpr float kWhole = 12582912.0f;
    const float inv = scale.s > 0.0f ? 1.0f / scale.s : 0.0f;
    float y[E], q[E], off = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        y[e] = x[e] * scale.up;
        q[e] = __builtin_fmaf(y[e], inv, kWhole);
        off = fmaxf(off, fabsf(__builtin_fmaf(y[e], inv, kWhole - q[e])));
    }
    if (off >= 0.5f - 0x1p-15f || scale.up > 1.0f) {   // the least scales are rounded so far that x / s passes 127
        const float half = 0.5f * scale.s;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float rest = __builtin_fmaf(kWhole - q[e], scale.s, y[e]), size = fabsf(rest);
            if (size > half || (size == half && (__builtin_bit_cast(uint32_t, q[e]) & 1) != 0)) q[e] += rest > 0.0f ? 1.0f : -1.0f;
            q[e] = fminf(fmaxf(q[e], kWhole - 127.0f), kWhole + 127.0f);
        }
    }
#pragma unroll
    for (int w = 0; w < E / 4; ++w) {
        const uint32_t b[4] = {__builtin_bit_cast(uint32_t, q[4 * w]), __builtin_bit_cast(uint32_t, q[4 * w + 1]),
                               __builtin_bit_cast(uint32_t, q[4 * w + 2]), __builtin_bit_cast(uint32_t, q[4 * w + 3])};
        words[w] = scale.s > 0.0f ? __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu) : 0u;
    }
}

using F32x2 = float __attribute__((ext_vector_type(2)));

/// The numbers of byte I's two codes, the low half's first.
template <int I>
__device__ __forceinline__ F32x2 numbersOf(uint32_t word) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, I);
}

/// codeFp4 of eight numbers, with a scale that is not NaN. x * inv, times
/// 1 - 2^-21 and 1 + 2^-21, lies on either side of x / s: where both round to the
/// same code, x / s does too, and where not, the border between the two codes,
/// times s, is compared as codeFp4 does.
__device__ __forceinline__ uint32_t codesFp4(const float (&x)[8], const Scale& scale) {
    const float inv = scale.s > 0.0f ? 1.0f / scale.s : 0.0f, under = inv * (1.0f - 0x1p-21f), over = inv * (1.0f + 0x1p-21f);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] * scale.up;
    uint32_t a = 0, b = 0;
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, y[0] * under, y[1] * under, 1.0f, 0);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(b, y[0] * over, y[1] * over, 1.0f, 0);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, y[2] * under, y[3] * under, 1.0f, 1);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(b, y[2] * over, y[3] * over, 1.0f, 1);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, y[4] * under, y[5] * under, 1.0f, 2);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(b, y[4] * over, y[5] * over, 1.0f, 2);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, y[6] * under, y[7] * under, 1.0f, 3);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(b, y[6] * over, y[7] * over, 1.0f, 3);
    if (a != b) {
        const F32x2 low[4] = {numbersOf<0>(a), numbersOf<1>(a), numbersOf<2>(a), numbersOf<3>(a)};
        const F32x2 high[4] = {numbersOf<0>(b), numbersOf<1>(b), numbersOf<2>(b), numbersOf<3>(b)};
        uint32_t past = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float border = 0.5f * (fabsf(low[e / 2][e % 2]) + fabsf(high[e / 2][e % 2]));
            const float rest = __builtin_fmaf(-border, scale.s, fabsf(y[e]));
            if (rest > 0.0f || (rest == 0.0f && (b >> 4 * e & 1) == 0)) past |= 15u << 4 * e;
        }
        a = (a & ~past) | (b & past);
    }
    return a;
}

}  // namespace mlk
