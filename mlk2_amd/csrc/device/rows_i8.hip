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

/// A wave a row, of any length and alignment: its largest magnitude, then its
/// codes.
template <typename T>
__global__ __launch_bounds__(256) void quantizeRowsAny(mlkd_quantize_rows p) {
    const int ln = threadIdx.x & 63;
    for (int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); r < p.rows; r += static_cast<int64_t>(gridDim.x) * 4) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        uint32_t top = 0;
        for (int64_t i = ln; i < p.cols; i += 64) top = max(top, mlk::magnitude(static_cast<float>(x[i])));
        const Scale s = mlk::scaleOf(waveMax(top), 127.0f);
        const float inv = 1.0f / s.s;
        int8_t* codes = p.codes + r * p.codes_stride;
        for (int64_t i = ln; i < p.cols; i += 64) codes[i] = static_cast<int8_t>(mlk::codeI8(static_cast<float>(x[i]), s, inv));
        if (ln == 0) p.scale[r] = s.stored;
    }
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

const char* mlkd_quantize_rows_kernel_name(const mlkd_quantize_rows* p) {
    static thread_local std::string name;
    name = std::string("quantizeRowsAny<") + typeName(p->dtype) + ">";
    return name.c_str();
}

int mlkd_launch_quantize_rows(const mlkd_quantize_rows* p, void* stream) {
    if (p->rows == 0) return 0;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p->rows + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? quantizeRowsAny<float> : p->dtype == MLKD_F16 ? quantizeRowsAny<_Float16> : quantizeRowsAny<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
