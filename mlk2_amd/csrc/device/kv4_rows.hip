// Heads of keys and values to and from the rows of a cache in 4 bits.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "bits.h"
#include "runtime_abi.h"

namespace {

using mlk::Scale;

/// Tokens that there are: those below the end of the last sequence.
__device__ __forceinline__ int64_t tokensOf(const mlkd_kv4_rows& p) {
    if (p.q_offsets == nullptr) return p.tokens;
    return max(int64_t{0}, min(p.tokens, static_cast<int64_t>(p.q_offsets[p.sequences])));
}

/// A wave a head of k or v, with any dim, strides and alignment, two elements a
/// lane and byte.
template <typename T, bool STORE>
__global__ __launch_bounds__(256) void kv4RowsAny(mlkd_kv4_rows p) {
    const int ln = threadIdx.x & 63, bytes = p.dim / 2;
    const int64_t heads = tokensOf(p) * p.kv_heads * 2;
    for (int64_t n = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); n < heads; n += static_cast<int64_t>(gridDim.x) * 4) {
        const bool value = (n & 1) != 0;
        const int64_t t = n / 2 / p.kv_heads;
        const int h = static_cast<int>(n / 2 % p.kv_heads);
        const int64_t row = p.slots != nullptr ? p.slots[t] : t;
        const bool held = row >= 0 && row < p.cache_rows;
        if (STORE && !held) continue;
        T* x = static_cast<T*>(value ? p.v : p.k) + t * (value ? p.v_stride : p.k_stride) + static_cast<int64_t>(h) * p.dim;
        uint8_t* codes = (value ? p.v_codes : p.k_codes) + row * (value ? p.v_codes_stride : p.k_codes_stride) + static_cast<int64_t>(h) * bytes;
        float* scale = (value ? p.v_scale : p.k_scale) + row * p.kv_heads + h;
        if constexpr (STORE) {
            float a[2][2] = {};
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ln + 64 * i >= bytes) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    a[i][e] = static_cast<float>(x[2 * (ln + 64 * i) + e]);
                    top = max(top, mlk::magnitude(a[i][e]));
                }
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
            const Scale s = mlk::scaleOf(top, 6.0f);
            const bool finite = top < 0x7f800000u;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ln + 64 * i < bytes) {
                    codes[ln + 64 * i] = finite ? static_cast<uint8_t>(mlk::codeFp4(a[i][0], s) | mlk::codeFp4(a[i][1], s) << 4) : uint8_t{0};
                }
            }
            if (ln == 0) *scale = s.stored;
        } else {
            if (!held) continue;
            const float s = *scale;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ln + 64 * i >= bytes) continue;
                const mlk::F32x2 v = mlk::numbersOf<0>(codes[ln + 64 * i]);
                x[2 * (ln + 64 * i)] = static_cast<T>(v[0] * s);
                x[2 * (ln + 64 * i) + 1] = static_cast<T>(v[1] * s);
            }
        }
    }
}

/// Eight elements a lane, LANES lanes a head of up to 8 LANES elements, of any
/// alignment: the heads of a token's k, then those of its v, side by side. A
/// head is read once and written once. Bound by memory: a store of 8191 tokens of
/// 8 heads of 128 in f16, 42 MB, takes 16 to 17 us and their load into f32, 76 MB,
/// 16; 64 tokens 3.6 and 2.9. x is asked for before its slot or the count of tokens
/// is known (what comes is dropped where those say so), which had it wait three
/// times. Two heads a thread in flight were as fast for many tokens and took 5.3 us
/// for 64.
template <typename T, int LANES, bool STORE>
__global__ __launch_bounds__(256) void kv4Rows(mlkd_kv4_rows p) {
    const int lane = threadIdx.x % LANES, c = lane * 8, bytes = p.dim / 2;
    const uint32_t heads = p.kv_heads, most = static_cast<uint32_t>(p.tokens) * 2 * heads, step = 256 / LANES;
    // A workgroup's lanes take as many turns, as their exchange asks.
    for (uint32_t n0 = blockIdx.x * step; n0 < most; n0 += gridDim.x * step) {
        const uint32_t own = n0 + threadIdx.x / LANES, n = min(own, most - 1), part = n / heads, h = n - part * heads, t = part >> 1;
        const bool value = (part & 1) != 0;
        T* x = static_cast<T*>(value ? p.v : p.k) + t * (value ? p.v_stride : p.k_stride) + static_cast<int64_t>(h) * p.dim + c;
        T raw[8] = {};
        if (STORE && c < p.dim) __builtin_memcpy(raw, x, sizeof(raw));
        const int64_t row = p.slots != nullptr ? p.slots[t] : static_cast<int64_t>(t);
        const bool held = own < static_cast<uint32_t>(tokensOf(p)) * 2 * heads && row >= 0 && row < p.cache_rows && c < p.dim;
        uint8_t* codes = (value ? p.v_codes : p.k_codes) + row * (value ? p.v_codes_stride : p.k_codes_stride) + static_cast<int64_t>(h) * bytes + c / 2;
        float* scale = (value ? p.v_scale : p.k_scale) + row * p.kv_heads + h;
        if constexpr (STORE) {
            float v[8];
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = static_cast<float>(raw[e]);
                top = max(top, mlk::magnitude(v[e]));
            }
#pragma unroll
            for (int d = LANES / 2; d > 0; d >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
            const Scale s = mlk::scaleOf(top, 6.0f);
            const uint32_t word = top < 0x7f800000u ? mlk::codesFp4(v, s) : 0u;
            if (held) {
                __builtin_memcpy(codes, &word, 4);
                if (lane == 0) *scale = s.stored;
            }
        } else if (held) {
            const float s = *scale;
            uint32_t word;
            __builtin_memcpy(&word, codes, 4);
            const mlk::F32x2 v[4] = {mlk::numbersOf<0>(word), mlk::numbersOf<1>(word), mlk::numbersOf<2>(word), mlk::numbersOf<3>(word)};
            T out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = static_cast<T>(v[e / 2][e % 2] * s);
            __builtin_memcpy(x, out, sizeof(out));
        }
    }
}

/// Whole lanes' elements, and heads that 32 bits count with a grid's more.
bool rowsApply(const mlkd_kv4_rows* p) { return p->dim % 8 == 0 && p->tokens * p->kv_heads < (int64_t{1} << 30); }

int lanesOf(const mlkd_kv4_rows* p) { return p->dim <= 32 ? 4 : p->dim <= 64 ? 8 : p->dim <= 128 ? 16 : 32; }

template <typename T, bool STORE>
void launchRows(const mlkd_kv4_rows* p, hipStream_t st) {
    const int lanes = lanesOf(p);
    const int64_t heads = p->tokens * p->kv_heads * 2, each = 256 / lanes;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((heads + each - 1) / each, int64_t{1} << 16)));
    auto* kernel = lanes == 4 ? kv4Rows<T, 4, STORE> : lanes == 8 ? kv4Rows<T, 8, STORE> : lanes == 16 ? kv4Rows<T, 16, STORE> : kv4Rows<T, 32, STORE>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, *p);
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

template <bool STORE>
const char* kernelName(const mlkd_kv4_rows* p) {
    static thread_local std::string name;
    name = rowsApply(p) ? std::string("kv4Rows<") + typeName(p->dtype) + ", " + std::to_string(lanesOf(p))
                        : std::string("kv4RowsAny<") + typeName(p->dtype);
    name += STORE ? ", true>" : ", false>";
    return name.c_str();
}

template <bool STORE>
int launch(const mlkd_kv4_rows* p, void* stream) {
    if (p->tokens == 0) return 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (rowsApply(p)) {
        p->dtype == MLKD_F32 ? launchRows<float, STORE>(p, st) : p->dtype == MLKD_F16 ? launchRows<_Float16, STORE>(p, st) : launchRows<__bf16, STORE>(p, st);
        return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
    }
    const int64_t heads = p->tokens * p->kv_heads * 2;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((heads + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? kv4RowsAny<float, STORE> : p->dtype == MLKD_F16 ? kv4RowsAny<_Float16, STORE> : kv4RowsAny<__bf16, STORE>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // namespace

extern "C" {

const char* mlkd_store_kv4_kernel_name(const mlkd_kv4_rows* p) { return kernelName<true>(p); }
const char* mlkd_load_kv4_kernel_name(const mlkd_kv4_rows* p) { return kernelName<false>(p); }
int mlkd_launch_store_kv4(const mlkd_kv4_rows* p, void* stream) { return launch<true>(p, stream); }
int mlkd_launch_load_kv4(const mlkd_kv4_rows* p, void* stream) { return launch<false>(p, stream); }

}  // extern "C"
