// Products of rows in 8-bit integers, with a scale for each row and column.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "runtime_abi.h"

namespace {

/// A thread an output, with any sizes, strides and alignment.
template <typename T>
__global__ __launch_bounds__(256) void matmulI8Any(mlkd_matmul_i8 p) {
    const int64_t total = p.m * p.n;
    for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t t = i / p.n, c = i % p.n;
        const int8_t *a = p.a + t * p.lda, *b = p.b + c * p.ldb;
        int sum = 0;
        for (int64_t k = 0; k < p.k; ++k) sum += static_cast<int>(a[k]) * b[k];
        float v = static_cast<float>(sum) * p.a_scale[t] * p.b_scale[c];
        if (p.bias != nullptr) v += p.bias[c];
        static_cast<T*>(p.out)[t * p.ldo + c] = static_cast<T>(v);
    }
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

int64_t mlkd_matmul_i8_work_bytes(const mlkd_matmul_i8*) { return 0; }

const char* mlkd_matmul_i8_kernel_names(const mlkd_matmul_i8* p) {
    static thread_local std::string name;
    name = std::string("matmulI8Any<") + typeName(p->dtype) + ">";
    return name.c_str();
}

int mlkd_launch_matmul_i8(const mlkd_matmul_i8* p, void* stream) {
    if (p->m == 0) return 0;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p->m * p->n + 255) / 256, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? matmulI8Any<float> : p->dtype == MLKD_F16 ? matmulI8Any<_Float16> : matmulI8Any<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
