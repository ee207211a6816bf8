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

template <int CTRL, int ROWS>
__device__ __forceinline__ int maxFrom(int v) {
    return max(v, __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false));
}

/// The largest value of a wave's lanes.
__device__ __forceinline__ int largest(int v) {
    v = maxFrom<0x111, 0xf>(v);   // rows of 16 lanes, from 1, 2, 4, 8 before
    v = maxFrom<0x112, 0xf>(v);
    v = maxFrom<0x114, 0xf>(v);
    v = maxFrom<0x118, 0xf>(v);
    v = maxFrom<0x142, 0xa>(v);   // the last lane of rows 0 and 2 to rows 1 and 3
    return __builtin_amdgcn_readlane(maxFrom<0x143, 0xc>(v), 63);   // lane 31 to rows 2 and 3
}

/// The rows from the smallest to the largest offset: all that a sequence holds,
/// as one sequence without keys. All lanes of a wave return the same.
__device__ __forceinline__ SeqSpan heldRows(const mlkd_attention& p) {
    int below = INT32_MIN, end = 0;   // ~ the smallest; the largest
    for (int i = threadIdx.x & 63; i <= p.sequences; i += 128) {   // two reads at a time
        const int a = p.q_offsets[i], b = p.q_offsets[min(i + 64, p.sequences)];
        below = max(below, max(~a, ~b));
        end = max(end, max(a, b));
    }
    const int64_t q1 = min(int64_t{largest(end)}, p.q_rows), q0 = min(max(int64_t{~largest(below)}, int64_t{0}), q1);
    return {q0, 0, static_cast<int32_t>(q1 - q0), 0};
}

__device__ __forceinline__ int32_t prefixOf(const mlkd_attention& p) {
    if (p.prefix_k == nullptr) return 0;
    if (p.prefix_len == nullptr) return static_cast<int32_t>(p.prefix_rows);
    return static_cast<int32_t>(min(max(static_cast<int64_t>(p.prefix_len[0]), int64_t{0}), p.prefix_rows));
}

}  // namespace mlk
