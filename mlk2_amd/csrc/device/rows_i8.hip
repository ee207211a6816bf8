// Rows in 8-bit integers with a scale each.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "bits.h"
#include "runtime_abi.h"

namespace {

using mlk::Scale;

__device__ __forceinline__ uint32_t waveMax(uint32_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d, 64)));
    return v;
}

/// N elements at `from`, of any alignment.
template <int N, typename T>
__device__ __forceinline__ void load(const T* from, float (&v)[N]) {
    T raw[N];
    __builtin_memcpy(raw, from, sizeof(raw));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(raw[i]);
}

/// A row to LANES threads, which hold it in registers, P pieces of 16 bytes each:
/// one read of x, one write of its codes. Rows and columns may have any
/// alignment; the last piece of a row may be a part of one. Bound by memory: 4096 rows
/// of 4096 in f16, 48 MB, take 15 us (by a wave a row, eight pieces each, 28), 64 of
/// them in bf16 4.8.
template <typename T, int LANES, int P>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void quantizeRows(mlkd_quantize_rows p) {
    constexpr int E = 16 / sizeof(T), BLOCK = LANES < 256 ? 256 : LANES, ROWS = BLOCK / LANES, WAVES = LANES / 64;
    __shared__ uint32_t tops[BLOCK / 64];
    const int lane = threadIdx.x % LANES;
    const int cols = static_cast<int>(p.cols);
    // All threads of a workgroup take as many turns, as the barriers ask.
    for (int64_t r0 = blockIdx.x * int64_t{ROWS}; r0 < p.rows; r0 += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t r = min(r0 + threadIdx.x / LANES, p.rows - 1);
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        float v[P][E];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * LANES + lane) * E;
            if (c + E <= cols) {
                load(x + c, v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[i][e] = c + e < cols ? static_cast<float>(x[c + e]) : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int e = 0; e < E; ++e) top = max(top, mlk::magnitude(v[i][e]));
        }
        top = waveMax(top);
        if constexpr (WAVES > 1) {
            if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top = max(top, tops[w]);
            __syncthreads();
        }
        const Scale s = mlk::scaleOf(top, 127.0f);
        int8_t* codes = p.codes + r * p.codes_stride;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * LANES + lane) * E;
            uint32_t words[E / 4];
            mlk::codesI8(v[i], s, words);
            int8_t q[E];
            __builtin_memcpy(q, words, E);
            if (c + E <= cols) {
                __builtin_memcpy(codes + c, q, E);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (c + e < cols) codes[c + e] = q[e];
                }
            }
        }
        if (lane == 0) p.scale[r] = s.stored;
    }
}

/// Rows longer than registers hold: a workgroup a row, which is read twice.
template <typename T>
__global__ __launch_bounds__(1024) void quantizeRowsLong(mlkd_quantize_rows p) {
    __shared__ uint32_t tops[16];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        uint32_t top = 0;
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) top = max(top, mlk::magnitude(static_cast<float>(x[i])));
        top = waveMax(top);
        if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 16; ++w) top = max(top, tops[w]);
        __syncthreads();
        const Scale s = mlk::scaleOf(top, 127.0f);
        const float inv = 1.0f / s.s;
        int8_t* codes = p.codes + r * p.codes_stride;
        for (int64_t i = threadIdx.x; i < p.cols; i += 1024) codes[i] = static_cast<int8_t>(mlk::codeI8(static_cast<float>(x[i]), s, inv));
        if (threadIdx.x == 0) p.scale[r] = s.stored;
    }
}

struct Plan {
    int lanes, pieces;   // 0 lanes: the long form
};

/// The fewest threads that hold a row in eight pieces each: a wave up to two, a
/// workgroup of four waves up to eight, one of sixteen beyond.
Plan planOf(const mlkd_quantize_rows* p) {
    const int64_t each = p->dtype == MLKD_F32 ? 4 : 8, pieces = (p->cols + each - 1) / each;
    if (pieces > 8 * 1024) return {0, 0};
    const int lanes = pieces <= 2 * 64 ? 64 : pieces <= 8 * 256 ? 256 : 1024;
    const int64_t per = (pieces + lanes - 1) / lanes;   // 256 lanes: above half a piece, 1024: above two
    return {lanes, lanes == 64 && per == 1 ? 1 : lanes != 1024 && per <= 2 ? 2 : per <= 4 ? 4 : 8};
}

template <typename T, int LANES, int P>
void launchRows(const mlkd_quantize_rows* p, hipStream_t st) {
    constexpr int block = LANES < 256 ? 256 : LANES, rows = block / LANES;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p->rows + rows - 1) / rows, int64_t{1} << 20)));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(quantizeRows<T, LANES, P>), grid, dim3(block), 0, st, *p);
}

template <typename T>
void launchPlan(const mlkd_quantize_rows* p, const Plan& n, hipStream_t st) {
    if (n.lanes == 0) {
        hipLaunchKernelGGL(quantizeRowsLong<T>, dim3(static_cast<unsigned>(std::min<int64_t>(p->rows, int64_t{1} << 20))), dim3(1024), 0, st, *p);
    } else if (n.lanes == 64) {
        n.pieces == 1 ? launchRows<T, 64, 1>(p, st) : launchRows<T, 64, 2>(p, st);
    } else if (n.lanes == 256) {
        n.pieces == 2 ? launchRows<T, 256, 2>(p, st) : n.pieces == 4 ? launchRows<T, 256, 4>(p, st) : launchRows<T, 256, 8>(p, st);
    } else {
        n.pieces == 4 ? launchRows<T, 1024, 4>(p, st) : launchRows<T, 1024, 8>(p, st);
    }
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

const char* mlkd_quantize_rows_kernel_name(const mlkd_quantize_rows* p) {
    static thread_local std::string name;
    const Plan n = planOf(p);
    if (n.lanes == 0) name = std::string("quantizeRowsLong<") + typeName(p->dtype) + ">";
    else name = std::string("quantizeRows<") + typeName(p->dtype) + ", " + std::to_string(n.lanes) + ", " + std::to_string(n.pieces) + ">";
    return name.c_str();
}

int mlkd_launch_quantize_rows(const mlkd_quantize_rows* p, void* stream) {
    if (p->rows == 0) return 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan n = planOf(p);
    p->dtype == MLKD_F32 ? launchPlan<float>(p, n, st) : p->dtype == MLKD_F16 ? launchPlan<_Float16>(p, n, st) : launchPlan<__bf16>(p, n, st);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
