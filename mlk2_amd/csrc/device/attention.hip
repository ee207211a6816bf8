// Attention over packed sequences, out = softmax(scale q k^T) v, with grouped
// heads, causal or not, keys in a cache, and optionally behind a prefix that
// all sequences share.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "attention_span.h"
#include "runtime_abi.h"

namespace {

using mlk::prefixOf;
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

/// A query row in one wave, with any strides and alignment: a lane per key for
/// the scores (f32 sums over d), then a lane per output column. The running
/// maximum and sum take one pass over the keys; only keys that the row sees
/// are read.
template <typename T>
__global__ __launch_bounds__(256) void attentionRows(mlkd_attention p) {
    const int ln = threadIdx.x & 63, d = p.dim, group = p.heads / p.kv_heads;
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4, rows = p.q_rows * p.heads;
    const float scale = static_cast<float>(p.scale * 1.4426950408889634);
    const int32_t np = prefixOf(p);
    for (int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); r < rows; r += waves) {
        const int64_t t = r / p.heads;
        const int h = static_cast<int>(r % p.heads), g = h / group;
        const int b = sequenceOf(p, t);
        if (b < 0) continue;
        const SeqSpan s = spanOf(p, b);
        const int32_t own = p.causal != 0
                                ? static_cast<int32_t>(max(int64_t{0}, min(int64_t{s.nk}, t - s.q0 + 1 + s.nk - s.nq)))
                                : s.nk;
        const T* qr = static_cast<const T*>(p.q) + t * p.q_stride + static_cast<int64_t>(h) * d;
        float q[4], acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = ln + 64 * i < d ? static_cast<float>(qr[ln + 64 * i]) * scale : 0.0f;
            acc[i] = 0.0f;
        }
        float m = -INFINITY, l = 0.0f;
        for (int part = 0; part < 2; ++part) {
            const int32_t n = part == 0 ? np : own;
            const int64_t ks = part == 0 ? p.prefix_k_stride : p.k_stride, vs = part == 0 ? p.prefix_v_stride : p.v_stride;
            const T* k = static_cast<const T*>(part == 0 ? p.prefix_k : p.k) + (part == 0 ? 0 : s.k0 * ks) + g * d;
            const T* v = static_cast<const T*>(part == 0 ? p.prefix_v : p.v) + (part == 0 ? 0 : s.k0 * vs) + g * d;
            for (int32_t j0 = 0; j0 < n; j0 += 64) {
                const int seen = min(64, n - j0);
                const T* kr = k + (j0 + min(ln, seen - 1)) * ks;
                float x = 0.0f;
                for (int c = 0; c < d; ++c) x += lane(c < 64 ? q[0] : c < 128 ? q[1] : c < 192 ? q[2] : q[3], c & 63) * static_cast<float>(kr[c]);
                if (ln >= seen) x = -INFINITY;
                const float top = fmaxf(m, waveMax(x));
                const float base = top == -INFINITY ? 0.0f : top;
                const float w = __builtin_amdgcn_exp2f(x - base), keep = __builtin_amdgcn_exp2f(m - base);
                l = l * keep + waveSum(w);
                m = top;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] *= keep;
                for (int j = 0; j < seen; ++j) {
                    const float wj = lane(w, j);
                    const T* vr = v + (j0 + j) * vs;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (ln + 64 * i < d) acc[i] += wj * static_cast<float>(vr[ln + 64 * i]);
                    }
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

int64_t mlkd_attention_work_bytes(const mlkd_attention*) { return 0; }

const char* mlkd_attention_kernel_names(const mlkd_attention* p) {
    static thread_local std::string name;
    name = std::string("attentionRows<") + typeName(p->dtype) + ">";
    return name.c_str();
}

int mlkd_launch_attention(const mlkd_attention* p, void* stream) {
    const int64_t rows = p->q_rows * p->heads;
    if (rows == 0) return 0;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? attentionRows<float> : p->dtype == MLKD_F16 ? attentionRows<_Float16> : attentionRows<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
