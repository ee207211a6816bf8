// The sequences of an attention launch as its kernels read them.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../device_abi.h"

namespace mlk {

/// One sequence's query rows and keys, clipped to the buffers.
struct SeqSpan {
    int64_t q0, k0;   // first query row, first key row
    int32_t nq, nk;
};

__device__ __forceinline__ SeqSpan spanOf(const mlkd_attention& p, int b) {
    SeqSpan s;
    const int64_t lo = min(max(static_cast<int64_t>(p.q_offsets[b]), int64_t{0}), p.q_rows);
    const int64_t hi = min(max(static_cast<int64_t>(p.q_offsets[b + 1]), lo), p.q_rows);
    s.q0 = lo;
    s.nq = static_cast<int32_t>(hi - lo);
    int64_t k0 = lo, nk = hi - lo;
    if (p.kv_start != nullptr) {
        k0 = p.kv_start[b];
        nk = k0 >= 0 && k0 < p.kv_rows ? min(static_cast<int64_t>(p.kv_len[b]), p.kv_rows - k0) : 0;
    }
    s.nk = static_cast<int32_t>(max(nk, int64_t{0}));
    s.k0 = s.nk > 0 ? k0 : 0;
    return s;
}

__device__ __forceinline__ int32_t prefixOf(const mlkd_attention& p) {
    if (p.prefix_k == nullptr) return 0;
    if (p.prefix_len == nullptr) return static_cast<int32_t>(p.prefix_rows);
    return static_cast<int32_t>(min(max(static_cast<int64_t>(p.prefix_len[0]), int64_t{0}), p.prefix_rows));
}

}  // namespace mlk
