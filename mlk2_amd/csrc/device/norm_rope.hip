// Head norms of q and k with the position rotation in the same pass, and the
// rows of k and v put into a cache.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "runtime_abi.h"

namespace {

/// The frequency of a pair in quarter turns per position, within 16 roundings.
__device__ __forceinline__ double quartersOf(const mlkd_norm_rope& p, int pair) {
    double f = 0.63661977236758134308;   // 2 / pi
#pragma unroll
    for (int k = 0; k < 7; ++k) f *= (pair >> k & 1) != 0 ? p.power[k] : 1.0;
    return f;
}

/// The cosine and sine of position `pos` at such a frequency. The quarter
/// turns are counted off in f64 (a position of 2^20 keeps 2^-29 of one, 2^31
/// 2^-18); the rest, at most half a quarter turn to either side, goes through
/// the Taylor sums of x = pi/2 r, |x| <= pi/4, whose next terms are x^11 / 11!
/// < 2e-9 and x^12 / 12! < 2e-10.
__device__ __forceinline__ void turn(double pos, double quarters, float& c, float& s) {
    const double a = pos * quarters, k = rint(a);
    const float x = static_cast<float>(a - k) * 1.5707963267948966f, x2 = x * x;
    float sn = x + x * x2 * (-1.6666667e-1f + x2 * (8.3333333e-3f + x2 * (-1.9841270e-4f + x2 * 2.7557319e-6f)));
    float cs = 1.0f + x2 * (-0.5f + x2 * (4.1666667e-2f + x2 * (-1.3888889e-3f + x2 * (2.4801587e-5f - x2 * 2.7557319e-7f))));
    const int q = static_cast<int>(k) & 3;   // below 2^31 2/pi quarter turns
    const float cq = (q & 1) != 0 ? sn : cs, sq = (q & 1) != 0 ? cs : sn;
    c = q == 1 || q == 2 ? -cq : cq;
    s = q >= 2 ? -sq : sq;
}

__device__ __forceinline__ int axisOf(const mlkd_norm_rope& p, int pair) {
    return pair < p.section_end[0] ? 0 : pair < p.section_end[1] ? 1 : 2;
}

__device__ __forceinline__ int64_t tokensOf(const mlkd_norm_rope& p) {
    if (p.q_offsets == nullptr) return p.tokens;
    return min(max(static_cast<int64_t>(p.q_offsets[p.sequences]), int64_t{0}), p.tokens);
}

/// Heads whose squares f32 does not hold: their sum is past its range, or mean
/// square and eps are below 2^-90 (squares lose bits from 2^-126 on, and
/// v_rsq_f32 takes what is below that for 0). The root is then taken of squares
/// of the elements times a power of two: 2^-70 (elements below 2^128 give
/// squares below 2^116) or 2^100 (elements below 2^-41 give squares below 2^118,
/// the smallest, 2^-149, 2^-98).
struct Rescale {
    float before, after;   // an element's factors, before and after the product with the root's inverse
    __device__ __forceinline__ float squares() const { return before * after; }
    __device__ __forceinline__ float eps(double e) const { return static_cast<float>(e * squares() * squares()); }
};
constexpr float kLeastSquare = 0x1p-90f;
__device__ __forceinline__ bool rescaled(float square) { return square < kLeastSquare || square == INFINITY; }
__device__ __forceinline__ Rescale rescaleOf(float square) {
    return {square < kLeastSquare ? 0x1p100f : 1.0f, square == INFINITY ? 0x1p-70f : 1.0f};
}

/// Orders the lanes' LDS accesses of one wave.
__device__ __forceinline__ void waveFence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/// A head per wave, any strides and alignment; pairs meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void normRopeHeads(mlkd_norm_rope p) {
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
            float square = sum / static_cast<float>(d) + static_cast<float>(p.eps);
            const bool far = rescaled(square);   // alike in all lanes
            const Rescale by = rescaleOf(square);
            if (far) {
                sum = 0.0f;
                for (int c = ln; c < d; c += 64) sum += y[c] * by.squares() * (y[c] * by.squares());
#pragma unroll
                for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
                square = sum / static_cast<float>(d) + by.eps(p.eps);
            }
            float r = 1.0f / sqrtf(square);
            if (far) {
                for (int c = ln; c < d; c += 64) y[c] = y[c] * by.before * r * by.after;
                r = 1.0f;
            }
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
                turn(p.positions[axisOf(p, pair) * p.tokens + t], quartersOf(p, pair), cs, sn);
                out = first ? out * cs - other * sn : out * cs + other * sn;
            }
            if (stored) o[c] = static_cast<T>(out);
        }
        waveFence();
    }
}

template <typename T>
using Vec8 = T __attribute__((ext_vector_type(8)));

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, true));
}

/// The value of lane i ^ 16.
__device__ __forceinline__ float across16(float v) {
    const int i = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 16) != 0 ? r[0] : r[1]);
}

/// The value of the lane LPH / 2 away in each group of LPH lanes, by register
/// permutations: quad swaps, mirrored halves, rotations in 16.
template <int LPH>
__device__ __forceinline__ float acrossHalf(float v) {
    if (LPH == 4) return dpp<0x4e>(v);                      // quad 2 3 0 1
    if (LPH == 8) return dpp<0x1b>(dpp<0x141>(v));          // half mirror, quad 3 2 1 0
    if (LPH == 16) return dpp<0x128>(v);                    // rotate by 8
    return across16(v);
}

/// The sum over a group of LPH lanes, in every lane.
template <int LPH>
__device__ __forceinline__ float groupSum(float v) {
    if (LPH <= 8) {
        v += dpp<0xb1>(v);                                  // quad 1 0 3 2
        v += dpp<0x4e>(v);
        return LPH == 8 ? v + dpp<0x141>(v) : v;
    }
    v += dpp<0x128>(v);
    v += dpp<0x124>(v);
    v += dpp<0x122>(v);
    v += dpp<0x121>(v);
    return LPH == 32 ? v + across16(v) : v;
}

/// LPH lanes a head, 8 columns each; `per` units of 64 / LPH heads a wave, all
/// of a token's where there are tokens enough: the angles, the same for every
/// head, are taken once and stay in registers. Memory bound: each value is
/// read and written once, 16 bytes a lane. Four units are read at a time, the
/// next four (or the next token's first) while these are worked on.
template <typename T, int LPH, bool INTERLEAVED>
__global__ __launch_bounds__(256, 4) void normRopeTokens(mlkd_norm_rope p, int per, int chunks) {
    using V = Vec8<T>;
    constexpr int HPW = 64 / LPH, PAIRS = INTERLEAVED ? 4 : 8, BATCH = sizeof(T) == 4 ? 2 : 4;
    const int ln = threadIdx.x & 63, at = ln % LPH, d0 = at * 8, sub = ln / LPH;
    const bool on = d0 < p.dim, turns = d0 < p.rot;
    const int half = p.rot / 2;
    const int unitsQ = (p.heads + HPW - 1) / HPW, unitsK = (p.kv_heads + HPW - 1) / HPW;
    const int units = unitsQ + (p.v != nullptr ? 2 : 1) * unitsK;
    const int waves = static_cast<int>(gridDim.x) * 4;
    const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
    const int u0 = w % chunks * per, u1 = min(u0 + per, units);   // waves is a multiple of chunks
    const int64_t n = tokensOf(p), step = waves / chunks;
    int64_t t = w / chunks;
    if (t >= n || u0 >= u1) return;
    struct Unit {
        int kind, h;   // q, k, v; this lane's head
    };
    auto unit = [&](int u) {
        const int kind = u < unitsQ ? 0 : u < unitsQ + unitsK ? 1 : 2;
        return Unit{kind, (u - (kind == 0 ? 0 : kind == 1 ? unitsQ : unitsQ + unitsK)) * HPW + sub};
    };
    auto load = [&](int64_t t, int u, V (&x)[BATCH]) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            x[i] = V{};
            if (u + i >= u1) continue;
            const auto [kind, h] = unit(u + i);
            const T* row = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                           t * (kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride);
            if (on && h < (kind == 0 ? p.heads : p.kv_heads)) x[i] = *reinterpret_cast<const V*>(row + h * p.dim + d0);
        }
    };
    V next[BATCH];
    load(t, u0, next);
    const bool normed = p.q_weight != nullptr;
    float wq[8], wk[8];
    if (on && normed && u0 < unitsQ + unitsK) {
        if (p.weight_dtype == MLKD_F32) {
            const Vec8<float> a = *reinterpret_cast<const Vec8<float>*>(static_cast<const float*>(p.q_weight) + d0);
            const Vec8<float> b = *reinterpret_cast<const Vec8<float>*>(static_cast<const float*>(p.k_weight) + d0);
#pragma unroll
            for (int j = 0; j < 8; ++j) wq[j] = a[j], wk[j] = b[j];
        } else {
            const V a = *reinterpret_cast<const V*>(static_cast<const T*>(p.q_weight) + d0);
            const V b = *reinterpret_cast<const V*>(static_cast<const T*>(p.k_weight) + d0);
#pragma unroll
            for (int j = 0; j < 8; ++j) wq[j] = static_cast<float>(a[j]), wk[j] = static_cast<float>(b[j]);
        }
    }
    const int partner = ln - at + (d0 < half ? at + half / 8 : at - half / 8);
    const bool full = p.rot == 8 * LPH;
    const float mean = 1.0f / static_cast<float>(p.dim), eps = static_cast<float>(p.eps);
    for (; t < n; t += step) {
        const int64_t slot = p.slots != nullptr ? p.slots[t] : t;
        float cs[PAIRS], sn[PAIRS];
        if (u0 < unitsQ + unitsK && turns) {
            const int pair0 = INTERLEAVED ? d0 / 2 : d0 < half ? d0 : d0 - half;
            double freq = quartersOf(p, pair0);
            int32_t pos = p.positions[t];
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                if (p.axes > 1) pos = p.positions[axisOf(p, pair0 + j) * p.tokens + t];
                turn(pos, freq, cs[j], sn[j]);
                if (!INTERLEAVED && d0 < half) sn[j] = -sn[j];
                freq *= p.power[0];
            }
        }
        for (int u = u0; u < u1; u += BATCH) {
            V x[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) x[i] = next[i];
            if (u + BATCH < u1) load(t, u + BATCH, next);
            else if (t + step < n) load(t + step, u0, next);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (u + i >= u1) break;
                const auto [kind, h] = unit(u + i);
                V z = x[i];
                if (kind < 2) {
                    float y[8], sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        y[j] = static_cast<float>(x[i][j]);
                        sum += y[j] * y[j];
                    }
                    if (normed) {
                        float square = groupSum<LPH>(sum) * mean + eps, r = __builtin_amdgcn_rsqf(square);
                        if (__any(rescaled(square))) {   // the other heads times 1
                            const Rescale by = rescaleOf(square);
                            sum = 0.0f;
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum += y[j] * by.squares() * (y[j] * by.squares());
                            r = __builtin_amdgcn_rsqf(groupSum<LPH>(sum) * mean + by.eps(p.eps));
#pragma unroll
                            for (int j = 0; j < 8; ++j) y[j] = y[j] * by.before * r * by.after;
                            r = 1.0f;
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = y[j] * r * (kind == 0 ? wq[j] : wk[j]);
                    }
                    if (INTERLEAVED) {
                        if (turns) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float e = y[2 * j], o = y[2 * j + 1];
                                y[2 * j] = e * cs[j] - o * sn[j];
                                y[2 * j + 1] = o * cs[j] + e * sn[j];
                            }
                        }
                    } else if (full) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = y[j] * cs[j] + acrossHalf<LPH>(y[j]) * sn[j];
                    } else if (p.rot > 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float other = __shfl(y[j], partner, 64);
                            if (turns) y[j] = y[j] * cs[j] + other * sn[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = static_cast<T>(y[j]);
                }
                const int64_t row = kind == 0 ? t : slot;
                T* out = static_cast<T*>(kind == 0 ? p.q_out : kind == 1 ? p.k_out : p.v_out) +
                         row * (kind == 0 ? p.q_out_stride : kind == 1 ? p.k_out_stride : p.v_out_stride);
                if (on && h < (kind == 0 ? p.heads : p.kv_heads) && (kind == 0 || (row >= 0 && row < p.out_rows))) {
                    *reinterpret_cast<V*>(out + h * p.dim + d0) = z;
                }
            }
        }
    }
}

/// Rows in whole 16-byte pieces, and pairs that are whole lanes' columns.
bool tokensApply(const mlkd_norm_rope* p) {
    const int e = 8, size = p->dtype == MLKD_F32 ? 4 : 2;
    auto aligned = [&](const void* ptr, int64_t stride) {
        return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && stride * size % 16 == 0;
    };
    const int weight = p->q_weight == nullptr || p->weight_dtype == p->dtype ? size : 4;
    if (p->q_weight != nullptr && (reinterpret_cast<uintptr_t>(p->q_weight) % (e * weight) != 0 ||
                                   reinterpret_cast<uintptr_t>(p->k_weight) % (e * weight) != 0)) {
        return false;
    }
    return p->dim % e == 0 && (p->interleaved ? p->rot % e == 0 : p->rot % (2 * e) == 0) && aligned(p->q, p->q_stride) &&
           aligned(p->k, p->k_stride) && aligned(p->v, p->v_stride) && aligned(p->q_out, p->q_out_stride) &&
           aligned(p->k_out, p->k_out_stride) && aligned(p->v_out, p->v_out_stride);
}

int lanesOf(const mlkd_norm_rope* p) { return p->dim <= 32 ? 4 : p->dim <= 64 ? 8 : p->dim <= 128 ? 16 : 32; }

template <typename T, bool INTERLEAVED>
void launchTokens(const mlkd_norm_rope& p, hipStream_t st) {
    const int lanes = lanesOf(&p), each = 64 / lanes;
    const int units = (p.heads + each - 1) / each + (p.v != nullptr ? 2 : 1) * ((p.kv_heads + each - 1) / each);
    // A token's units in one wave, or spread over several until the chip has
    // its four waves a SIMD; waves take tokens in turn (8192 tokens of 48 heads
    // of 128: 44.0 us, 4.57 TB/s, with 4096 waves, 44.0 with 8192, 49.5 with
    // 16384, 53.2 with 2048; 4099 of 48 of 64: 16.1, 17.6, 21.1, 20.1).
    constexpr int64_t kWaves = 4096;
    const int most = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(units, kWaves / p.tokens)));
    const int per = (units + most - 1) / most, chunks = (units + per - 1) / per;
    const int64_t want = std::min<int64_t>(p.tokens * chunks, kWaves), unit = 4 * chunks;   // whole tokens, whole workgroups
    const dim3 grid(static_cast<unsigned>((want + unit - 1) / unit * chunks));
    auto* kernel = lanes == 4    ? normRopeTokens<T, 4, INTERLEAVED>
                   : lanes == 8  ? normRopeTokens<T, 8, INTERLEAVED>
                   : lanes == 16 ? normRopeTokens<T, 16, INTERLEAVED>
                                 : normRopeTokens<T, 32, INTERLEAVED>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, per, chunks);
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

const char* mlkd_norm_rope_kernel_name(const mlkd_norm_rope* p) {
    static thread_local std::string name;
    name = std::string("normRopeHeads<") + typeName(p->dtype) + ">";
    if (tokensApply(p)) {
        name = std::string("normRopeTokens<") + typeName(p->dtype) + ", " + std::to_string(lanesOf(p)) +
               (p->interleaved != 0 ? ", true>" : ", false>");
    }
    return name.c_str();
}

int mlkd_launch_norm_rope(const mlkd_norm_rope* p, void* stream) {
    if (p->tokens == 0) return 0;
    if (tokensApply(p)) {
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const bool inter = p->interleaved != 0;
        if (p->dtype == MLKD_F32) inter ? launchTokens<float, true>(*p, st) : launchTokens<float, false>(*p, st);
        else if (p->dtype == MLKD_F16) inter ? launchTokens<_Float16, true>(*p, st) : launchTokens<_Float16, false>(*p, st);
        else inter ? launchTokens<__bf16, true>(*p, st) : launchTokens<__bf16, false>(*p, st);
        return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
    }
    const int64_t heads = p->tokens * (p->heads + 2 * p->kv_heads);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((heads + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? normRopeHeads<float> : p->dtype == MLKD_F16 ? normRopeHeads<_Float16> : normRopeHeads<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
