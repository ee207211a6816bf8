// Attention over packed sequences whose keys and values are a cache's in 4 bits.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "attention_span.h"
#include "bits.h"
#include "runtime_abi.h"

namespace {

using mlk::SeqSpan;
using mlk::spanOf;

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

/// The sequence that holds query row t, or -1.
__device__ __forceinline__ int sequenceOf(const mlkd_attention& p, int64_t t) {
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.q_offsets[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && t < p.q_offsets[lo] ? lo - 1 : -1;
}

/// A query row in one wave, with any even dim, strides and alignment: a lane per
/// key for the scores, then a lane per output column.
template <typename T>
__global__ __launch_bounds__(256) void attentionKv4Rows(mlkd_attention_kv4 args) {
    const mlkd_attention& p = args.a;
    const int ln = threadIdx.x & 63, d = p.dim, group = p.heads / p.kv_heads;
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4, rows = p.q_rows * p.heads;
    const float scale = static_cast<float>(p.scale * 1.4426950408889634);
    for (int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); r < rows; r += waves) {
        const int64_t t = r / p.heads;
        const int h = static_cast<int>(r % p.heads), g = h / group;
        const int b = sequenceOf(p, t);
        if (b < 0) continue;
        const SeqSpan s = spanOf(p, b);
        const int64_t own = p.causal != 0 ? max(int64_t{0}, min(int64_t{s.nk}, t - s.q0 + 1 + s.nk - s.nq)) : s.nk;
        const T* qr = static_cast<const T*>(p.q) + t * p.q_stride + static_cast<int64_t>(h) * d;
        float q[4], acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = ln + 64 * i < d ? static_cast<float>(qr[ln + 64 * i]) : 0.0f;
            acc[i] = 0.0f;
        }
        auto query = [&](int c) { return lane(c < 64 ? q[0] : c < 128 ? q[1] : c < 192 ? q[2] : q[3], c & 63); };
        float m = -INFINITY, l = 0.0f;
        const uint8_t* k = static_cast<const uint8_t*>(p.k) + s.k0 * p.k_stride + g * (d / 2);
        const uint8_t* v = static_cast<const uint8_t*>(p.v) + s.k0 * p.v_stride + g * (d / 2);
        for (int64_t j0 = 0; j0 < own; j0 += 64) {
            const int seen = static_cast<int>(min(int64_t{64}, own - j0));
            const int64_t j = j0 + min(ln, seen - 1), at = (s.k0 + j) * p.kv_heads + g;
            const uint8_t* kr = k + j * p.k_stride;
            float x = 0.0f;
            for (int c = 0; c < d / 2; ++c) {
                const mlk::F32x2 n = mlk::numbersOf<0>(kr[c]);
                x += query(2 * c) * n[0];
                x += query(2 * c + 1) * n[1];
            }
            x *= args.k_scale[at] * scale;
            const float vs = args.v_scale[at];
            if (ln >= seen) x = -INFINITY;
            const float top = fmaxf(m, waveMax(x));
            const float base = top == -INFINITY ? 0.0f : top;
            const float w = __builtin_amdgcn_exp2f(x - base), keep = __builtin_amdgcn_exp2f(m - base);
            l = l * keep + waveSum(w);
            m = top;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= keep;
            for (int i = 0; i < seen; ++i) {
                const float wi = lane(w, i) * lane(vs, i);
                const uint8_t* vr = v + (j0 + i) * p.v_stride;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int c = ln + 64 * n;
                    if (c < d) acc[n] += wi * mlk::numbersOf<0>(vr[c >> 1] >> (c & 1) * 4)[0];
                }
            }
        }
        // A sum of no weights; one that is NaN stays one.
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* o = static_cast<T*>(p.out) + t * p.out_stride + static_cast<int64_t>(h) * d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ln + 64 * i < d) o[ln + 64 * i] = static_cast<T>(acc[i] * inv);
        }
        if (p.lse != nullptr && ln == 0) p.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

int64_t mlkd_attention_kv4_work_bytes(const mlkd_attention_kv4*) { return 0; }

const char* mlkd_attention_kv4_kernel_names(const mlkd_attention_kv4* p) {
    static thread_local std::string name;
    name = std::string("attentionKv4Rows<") + typeName(p->a.dtype) + ">";
    return name.c_str();
}

int mlkd_launch_attention_kv4(const mlkd_attention_kv4* p, void* stream) {
    const int64_t rows = p->a.q_rows * p->a.heads;
    if (rows == 0) return 0;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->a.dtype == MLKD_F32 ? attentionKv4Rows<float> : p->a.dtype == MLKD_F16 ? attentionKv4Rows<_Float16> : attentionKv4Rows<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
