// What attention's kernels have alike beside their tiles: a row's sequence, the
// join of key ranges. For inclusion in one source each.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "attention_tiles.h"

namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float waveMax(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

__device__ __forceinline__ float waveSum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ float lane(float v, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}

/// The sequence that holds query row t, or -1: the last whose first row is at
/// or before it, where that one reaches it.
__device__ __forceinline__ int sequenceOf(const mlkd_attention& p, int64_t t) {
    int lo = 0, hi = p.sequences;   // q_offsets[lo - 1] <= t < q_offsets[hi], as far as they are in order
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.q_offsets[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && t < p.q_offsets[lo] ? lo - 1 : -1;
}

/// The results of key ranges joined: out = sum acc_i 2^(m_i - m) / sum l_i
/// 2^(m_i - m), m the largest maximum. A wave a row, LPR lanes to a range with 4
/// columns each, so that ranges are read side by side, four of them in flight.
/// Bound by the waits of a row's few dependent reads: 2048 rows of 128 columns
/// and 17 ranges in 6.7 us (18 MB), 11688 rows of 64 and 5 ranges in 9.3.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void attentionJoin(mlk::TileArgs a) {
    const mlkd_attention& p = a.p;
    using mlk::f32x4;
    constexpr int SIDE = 64 / LPR;
    const int ln = threadIdx.x & 63, column = ln % LPR * 4;
    const int64_t rows = p.q_rows * p.heads;
    for (int64_t r = blockIdx.x * int64_t{4} + threadIdx.x / 64; r < rows; r += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t t = rows < (int64_t{1} << 30) ? static_cast<int>(r) / a.by_heads : r / p.heads;
        // A row of no sequence is left alone.
        bool held = false;
        for (int s = ln; s < p.sequences; s += 64) held |= p.q_offsets[s] <= t && t < p.q_offsets[s + 1];
        // The weights of the ranges, lane i those of i and 64 + i; below 0: a
        // range without keys, its sums may not have been written.
        float2 ml[2];
        float w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) ml[h] = ln + 64 * h < a.parts ? a.ml[(ln + 64 * h) * rows + r] : make_float2(mlk::kLowest, 0.0f);
        if (!__any(held)) continue;
        const float m = waveMax(fmaxf(ml[0].x, ml[1].x));
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = __builtin_amdgcn_exp2f(ml[h].x - m);
        const float l = waveSum(ml[0].y * w[0] + ml[1].y * w[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = ml[h].y == 0.0f ? -1.0f : w[h];
        f32x4 sum = {};
        const float* from = a.acc + r * p.dim + column;
#pragma unroll 1
        for (int i0 = 0; i0 < a.parts; i0 += 4 * SIDE) {
            f32x4 v[4];
            float u[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = i0 + n * SIDE + ln / LPR;
                u[n] = __shfl(i0 + n * SIDE < 64 ? w[0] : w[1], i & 63);
                v[n] = f32x4{};
                if (i < a.parts && u[n] >= 0.0f && column < p.dim) v[n] = *reinterpret_cast<const f32x4*>(from + i * rows * p.dim);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) sum += fmaxf(u[n], 0.0f) * v[n];
        }
#pragma unroll
        for (int d = LPR; d < 64; d *= 2) {
#pragma unroll
            for (int f = 0; f < 4; ++f) sum[f] += __shfl_xor(sum[f], d);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (column < p.dim && ln < LPR) {
            mlk::Vec4<T> v;
#pragma unroll
            for (int f = 0; f < 4; ++f) v[f] = static_cast<T>(sum[f] * inv);
            *reinterpret_cast<mlk::Vec4<T>*>(static_cast<T*>(p.out) + t * p.out_stride + (r % p.heads) * p.dim + column) = v;
        }
        if (p.lse != nullptr && ln == 0) p.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

bool aligned(const void* ptr, int64_t stride, int bytes, int size) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && stride * size % bytes == 0 && stride < (int64_t{1} << 22);
}

mlk::Divider dividerOf(int d) {
    if (d == 1) return {0, 0};
    int up = 0;
    while ((int64_t{1} << up) < d) ++up;
    return {static_cast<uint32_t>(((uint64_t{1} << (31 + up)) + d - 1) / d), up - 1};
}

}  // namespace
