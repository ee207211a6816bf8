// Head norms of q and k with the position rotation in the same pass, and the
// rows of k and v put into a cache.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "runtime_abi.h"

namespace {

/// The cosine and sine of position `pos` at a frequency given in quarter turns
/// per position. The quarter turns are counted off in f64, where positions of
/// any i32 keep 2^-22 of one; the rest, at most half a quarter turn to either
/// side, goes through the Taylor sums of x = pi/2 r, |x| <= pi/4, whose next
/// terms are x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10.
__device__ __forceinline__ void turn(double pos, double quarters, float& c, float& s) {
    const double a = pos * quarters, k = rint(a);
    const float x = static_cast<float>(a - k) * 1.5707963267948966f, x2 = x * x;
    float sn = x + x * x2 * (-1.6666667e-1f + x2 * (8.3333333e-3f + x2 * (-1.9841270e-4f + x2 * 2.7557319e-6f)));
    float cs = 1.0f + x2 * (-0.5f + x2 * (4.1666667e-2f + x2 * (-1.3888889e-3f + x2 * (2.4801587e-5f - x2 * 2.7557319e-7f))));
    const int q = static_cast<int>(k - 4.0 * floor(k * 0.25));   // 0 .. 3
    const float cq = (q & 1) != 0 ? sn : cs, sq = (q & 1) != 0 ? cs : sn;
    c = q == 1 || q == 2 ? -cq : cq;
    s = q >= 2 ? -sq : sq;
}

/// Kernel arguments: the descriptor and the frequency of each pair.
struct NormRopeArgs {
    mlkd_norm_rope p;
    double quarters[128];
};

__device__ __forceinline__ int axisOf(const mlkd_norm_rope& p, int pair) {
    return pair < p.section_end[0] ? 0 : pair < p.section_end[1] ? 1 : 2;
}

__device__ __forceinline__ int64_t tokensOf(const mlkd_norm_rope& p) {
    if (p.q_offsets == nullptr) return p.tokens;
    return min(max(static_cast<int64_t>(p.q_offsets[p.sequences]), int64_t{0}), p.tokens);
}

/// Orders the lanes' LDS accesses of one wave.
__device__ __forceinline__ void waveFence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/// A head per wave, any strides and alignment; pairs meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void normRopeHeads(NormRopeArgs a) {
    const mlkd_norm_rope& p = a.p;
    __shared__ float ys[4][256];
    float* y = ys[threadIdx.x >> 6];
    const int ln = threadIdx.x & 63, d = p.dim, half = p.rot / 2;
    const int heads = p.heads + (p.v != nullptr ? 2 : 1) * p.kv_heads;
    const int64_t n = tokensOf(p) * heads, waves = static_cast<int64_t>(gridDim.x) * 4;
    for (int64_t i = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); i < n; i += waves) {
        const int64_t t = i / heads;
        int h = static_cast<int>(i % heads);
        const int kind = h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;   // q, k, v
        h -= kind == 0 ? 0 : kind == 1 ? p.heads : p.heads + p.kv_heads;
        const T* x = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                     t * (kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride) + static_cast<int64_t>(h) * d;
        const int64_t row = kind == 0 || p.slots == nullptr ? t : p.slots[t];
        const bool stored = kind == 0 || (row >= 0 && row < p.out_rows);
        T* o = static_cast<T*>(kind == 0 ? p.q_out : kind == 1 ? p.k_out : p.v_out) +
               (stored ? row : 0) * (kind == 0 ? p.q_out_stride : kind == 1 ? p.k_out_stride : p.v_out_stride) +
               static_cast<int64_t>(h) * d;
        float sum = 0.0f;
        for (int c = ln; c < d; c += 64) {
            y[c] = static_cast<float>(x[c]);
            sum += y[c] * y[c];
        }
        if (kind < 2 && p.q_weight != nullptr) {
#pragma unroll
            for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
            const float r = 1.0f / sqrtf(sum / static_cast<float>(d) + static_cast<float>(p.eps));
            const void* w = kind == 0 ? p.q_weight : p.k_weight;
            for (int c = ln; c < d; c += 64) {
                y[c] = y[c] * r * (p.weight_dtype == MLKD_F32 ? static_cast<const float*>(w)[c] : static_cast<float>(static_cast<const T*>(w)[c]));
            }
        }
        waveFence();
        for (int c = ln; c < d; c += 64) {
            float out = y[c];
            if (kind < 2 && c < p.rot) {
                const int pair = p.interleaved ? c / 2 : c < half ? c : c - half;
                const bool first = p.interleaved ? c % 2 == 0 : c < half;
                const float other = y[p.interleaved ? c ^ 1 : first ? c + half : c - half];
                float cs, sn;
                turn(p.positions[axisOf(p, pair) * p.tokens + t], a.quarters[pair], cs, sn);
                out = first ? out * cs - other * sn : out * cs + other * sn;
            }
            if (stored) o[c] = static_cast<T>(out);
        }
        waveFence();
    }
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

const char* mlkd_norm_rope_kernel_name(const mlkd_norm_rope* p) {
    static thread_local std::string name;
    name = std::string("normRopeHeads<") + typeName(p->dtype) + ">";
    return name.c_str();
}

int mlkd_launch_norm_rope(const mlkd_norm_rope* p, void* stream) {
    if (p->tokens == 0) return 0;
    NormRopeArgs a;
    a.p = *p;
    for (int i = 0; i < 128; ++i) a.quarters[i] = i < p->rot / 2 ? p->quarters[i] : 0.0;
    const int64_t heads = p->tokens * (p->heads + 2 * p->kv_heads);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((heads + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? normRopeHeads<float> : p->dtype == MLKD_F16 ? normRopeHeads<_Float16> : normRopeHeads<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
