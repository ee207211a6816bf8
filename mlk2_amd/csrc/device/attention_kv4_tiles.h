// Attention over a cache in 4 bits on matrix cores: a wave 16 or 32 query rows,
// over tiles of 32 keys.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "attention_tiles.h"

namespace mlk {

using i32x2 = int __attribute__((ext_vector_type(2)));
using i32x4 = int __attribute__((ext_vector_type(4)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));

struct Kv4Args {
    TileArgs t;                      // p's k and v: the codes, strides in bytes
    const float *k_scale, *v_scale;  // [kv_rows, kv_heads]
    int units;                       // row blocks, or with parts their key ranges, of one head at most
    // scale log2 e = c codes 2^up, c below 2 in size, so that a key's scale times c is in
    // range: the keys' codes are taken times `codes`, 2^13 at most, the queries times 2^up.
    float c, codes;
    int up;
};

/// The numbers of a word's eight codes times a power of two, exact in either type (f16:
/// up to 2^13).
template <typename T>
__device__ __forceinline__ Piece<T> numbers(int word, float by);
template <>
__device__ __forceinline__ Piece<__bf16> numbers<__bf16>(int word, float by) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, by, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, by, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, by, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, by, 3);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
template <>
__device__ __forceinline__ Piece<_Float16> numbers<_Float16>(int word, float by) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, by, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, by, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, by, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, by, 3);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int N>
using F32 = float __attribute__((ext_vector_type(N)));

/// c += a b: 32 x 32 by 16, or 16 x 16 by 32.
template <int EDGE>
__device__ __forceinline__ F32<EDGE * EDGE / 64> product(Piece<__bf16> a, Piece<__bf16> b, F32<EDGE * EDGE / 64> c) {
    if constexpr (EDGE == 32) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <int EDGE>
__device__ __forceinline__ F32<EDGE * EDGE / 64> product(Piece<_Float16> a, Piece<_Float16> b, F32<EDGE * EDGE / 64> c) {
    if constexpr (EDGE == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/// The value of lane l ^ 16.
__device__ __forceinline__ float otherSixteen(float v) {
    const int i = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 16) != 0 ? r[0] : r[1]);
}

/// The largest, and the sum, over the lanes of one query: those EDGE apart.
template <int EDGE>
__device__ __forceinline__ float largestOf(float v) {
    if constexpr (EDGE == 16) v = fmaxf(v, otherSixteen(v));
    return fmaxf(v, otherHalf(v));
}
template <int EDGE>
__device__ __forceinline__ float sumOf(float v) {
    if constexpr (EDGE == 16) v += otherSixteen(v);
    return v + otherHalf(v);
}

/// Whether some of the queries that a lane takes, eight at a time, may be too far from
/// one for sums of them times codes, or for their parts.
template <typename T>
struct Sizes;
template <>
struct Sizes<__bf16> {
    float squares[2] = {};
    __device__ __forceinline__ void take(Piece<__bf16> v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16x2 two = {v[2 * i], v[2 * i + 1]};
            squares[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(two, two, squares[i & 1], false);
        }
    }
    __device__ __forceinline__ bool far() const { return squares[0] + squares[1] > 0x1p120f; }
};
template <>
struct Sizes<_Float16> {
    __device__ __forceinline__ void take(Piece<_Float16>) {}
    __device__ __forceinline__ bool far() const { return false; }
};
template <>
struct Sizes<float> {
    float top = 0.0f;
    __device__ __forceinline__ void take(float __attribute__((ext_vector_type(8))) v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    }
    __device__ __forceinline__ bool far() const { return top > 0.0f && !(top >= 0x1p-60f && top <= 0x1p100f); }
};

/// NW waves with the same ROWS query rows, tiles of 32 keys in turn; their sums are
/// joined at the end.
template <typename T, int DT, int ROWS, int NW>
struct Kv4Tiles {
    using Q = std::conditional_t<std::is_same_v<T, float>, __bf16, T>;      // the scores' operands
    static constexpr int kPartsQ = std::is_same_v<T, float> ? 3 : 1;        // of a query: 24 bits in 8 each
    static constexpr int kPartsW = std::is_same_v<T, float> ? 3 : std::is_same_v<T, _Float16> ? 2 : 1;   // of a weight
    static constexpr int kEdge = ROWS < 32 ? 16 : 32, kLanes = 64 / kEdge;  // of a product; lanes of a query (or a key)
    static constexpr int QB = ROWS / kEdge, KB = 32 / kEdge;                // blocks of queries, of a tile's keys
    static constexpr int KS = DT / 8 / kLanes;                              // steps of q k^T, eight elements a lane
    static constexpr int NS = kEdge * kEdge / 64 * KB;                      // scores of a lane, per block of queries
    static constexpr int NO = kEdge * kEdge / 64, DB = DT / kEdge;          // sums of a lane and block of out; its blocks
    static constexpr int kPieces = DT <= 64 ? 2 : DT <= 128 ? 4 : 8;        // 16-byte pieces of a row in LDS
    static constexpr int kPitch = 16 * kPieces;
    static constexpr int kHalf = 32 * kPitch, kStage = 2 * kHalf + 256;     // a tile's keys (or values); with the scales
    static constexpr int kLoads = kHalf / 1024;                             // of 64 pieces, for keys and again for values
    static constexpr int kPerTile = 2 * kLoads + 1;
    static constexpr int kStages = 3;                                       // three times four waves fit a compute unit
    static constexpr int kRing = kStage * kStages;
    static constexpr int kRow = DT * 4;                                     // bytes of a row of results
    static constexpr int kJoin = 16 * (kRow + 8);                           // sixteen rows at a time
    static constexpr int kLds = NW * (kRing > kJoin ? kRing : kJoin);
    static_assert(kPerTile * (kStages - 1) <= 63, "the loads waited on by number fit the counter");
    // Exponents between which a row's largest query is left as it is: sums of 256 of
    // them times 6 2^13 stay in f32's range, and the last of three bf16 parts in bf16's.
    // f16 itself holds less.
    static constexpr int kLeast = std::is_same_v<T, _Float16> ? -24 : -60, kMost = std::is_same_v<T, _Float16> ? 16 : 103;

    /// Turn of row j's pieces, so that the rows that are read at a time lie in
    /// different banks: 16 from one on, or fours of them eight or sixteen apart.
    static __device__ __forceinline__ int swizzle(int j) {
        return kPieces == 2 ? j >> 3 & 1 : kPieces == 4 ? (j >> 2 & 3) ^ (j >> 4 & 1) : (j >> 1 & 7) ^ (j >> 4 & 1) << 1;
    }

    /// 16 (or 4) bytes a lane to LDS at `m0` + 16 (4) * lane. A load to LDS takes M0
    /// one wait state after a scalar write of it at the earliest (s_nop 0).
    static __device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t m0) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
    }
    static __device__ __forceinline__ void dma4(const void* from, uint32_t m0) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
    }
    /// Waits until at most `ahead` tiles of this wave's loads are in flight, and no
    /// read of LDS.
    static __device__ __forceinline__ void wait(int ahead) {
        static_assert(kStages == 3, "");
        if (ahead >= 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kPerTile) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
};

/// What a workgroup takes: a row block of a sequence, and which of so many ranges of
/// its keys.
struct Kv4Unit {
    SeqSpan s;
    int r0, split, splits;
};

/// Unit `unit` of `units`, which are dealt out by the keys there are: a sequence's
/// row blocks are split into as many ranges, `parts` at most, as make all of them
/// about equally long, so that all units of a launch run at once and end together
/// (32 single tokens over 1000 to 8192 keys 51.7 us, whole 60.9). For 64 sequences at
/// most, a lane each, and more units than there are row blocks.
template <int ROWS>
__device__ __forceinline__ bool dealtUnit(const mlkd_attention& p, int group, int unit, int units, int parts, Kv4Unit& u) {
    const int ln = threadIdx.x & 63;
    SeqSpan of{};
    if (ln < p.sequences) of = spanOf(p, ln);
    const int blocks = (of.nq * group + ROWS - 1) / ROWS, tiles = blocks > 0 ? (of.nk + 31) / 32 : 0;
    const int free = units - __builtin_amdgcn_readlane(sumUpTo(blocks), 63);   // units beside a block's first
    float all = static_cast<float>(blocks) * static_cast<float>(tiles);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d, 64);
    // The shortest range that the units suffice for, to a sixteenth of where it lies:
    // no shorter than all tiles over all units, and all over the free ones (a little
    // more than exactly) has room for the blocks' last, shorter ranges. One tile for
    // each wave at least, two where the ranges' number is no limit.
    const int shortest = max(8, (largest(tiles) + parts - 1) / parts);
    auto rangesOf = [&](int range) { return max(1, (tiles + range - 1) / range); };
    int range = max(shortest, static_cast<int>(fminf(all / static_cast<float>(free) * 1.001f, 1e9f)) + 1);
    int below = max(shortest, static_cast<int>(fminf(all / static_cast<float>(units), 1e9f)));
    for (int n = 0; n < 4 && below < range; ++n) {
        const int middle = (below + range) / 2;
        if (__builtin_amdgcn_readlane(sumUpTo(blocks * rangesOf(middle)), 63) <= units) range = middle;
        else below = middle + 1;
    }
    const int ranges = rangesOf(range);
    const int sum = sumUpTo(blocks * ranges);
    const uint64_t past = __ballot(sum > unit);
    if (past == 0) return false;
    const int b = __builtin_ctzll(past), at = unit - __builtin_amdgcn_readlane(sum - blocks * ranges, b);
    u.splits = __builtin_amdgcn_readlane(ranges, b);
    const int block = at / u.splits;
    u.split = at - block * u.splits;
    u.r0 = (__builtin_amdgcn_readlane(blocks, b) - 1 - block) * ROWS;
    u.s = SeqSpan{laneOf(of.q0, b), laneOf(of.k0, b), __builtin_amdgcn_readlane(of.nq, b), __builtin_amdgcn_readlane(of.nk, b)};
    return true;
}

/// Waves of a SIMD that the registers have to hold. f32 rows by 32 of dims up to 96
/// keep to 256 registers with it (3 x 129 of dim 64 over 777 12.9 us, 14.0 without; 2
/// x 500 of 96 over 1000 44.6, and 68.3 with one wave); of 256 they spill 35.
template <typename T>
constexpr int kv4Waves(int dt, int rows) {
    return rows == 16 ? (std::is_same_v<T, float> || dt > 128 ? 2 : 3) : dt > (std::is_same_v<T, float> ? 96 : 128) ? 1 : 2;
}

/// One row block of one key/value head. With S^T = K Q^T a lane holds some keys'
/// scores of one query, so the softmax is register work but for one exchange of
/// maxima. Prompts are bound by the wave's vector instructions and products, which
/// overlap little (1700 cycles for 32 rows and keys of 128; 4 prompts of 125 to 1000
/// tokens behind up to 4000, 32 heads on 8: 204 us, 0.69 PFLOP/s, matrix units busy in
/// 0.31 of the units' cycles), single tokens by memory and the start, 5 us to a first
/// tile's sums (32 over 1000 to 8192 keys, 165 MB: 47 us; all of 8192, whole, 285 MB:
/// 69, 4.1 TB/s). The products run on the codes as numbers, which either
/// 16-bit type holds exactly: a key's scale goes to its scores, a value's to its
/// weights. Codes come
/// straight to LDS, two tiles ahead; a word of a key's row is eight elements of
/// the product's operand as it lies. Values are read transposed, 4 bits at a time:
/// a lane gets a column's numbers of the keys whose weights it holds, in their
/// order.
///
/// What is rounded: a weight times its value's scale to bf16 (f16 rows: to two
/// bf16 parts, 16 bits, f32 rows three), half a step of itself or, below 2^-126,
/// 2^-134; f32 queries are three bf16 parts, exactly down to 2^-50 of the row's largest.
/// Scores, weights, their sum and out's sums are f32.
/// The maximum that the weights are relative to follows the running one only when
/// that has grown by 2^8.
template <typename T, int DT, int ROWS, int NW>
__global__ __launch_bounds__(NW * 64, kv4Waves<T>(DT, ROWS)) void attentionKv4Tiles(Kv4Args args) {
    using S = Kv4Tiles<T, DT, ROWS, NW>;
    using Q = typename S::Q;
    constexpr int EDGE = S::kEdge, QB = S::QB, KB = S::KB, KS = S::KS, NS = S::NS, NO = S::NO, DB = S::DB;
    extern __shared__ __align__(16) char ldsTiles[];
    const TileArgs& a = args.t;
    const mlkd_attention& p = a.p;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int ln = threadIdx.x & 63, col = ln % EDGE, part = ln / EDGE;
    // The heads of a unit go to one XCD one after the other: neighbouring heads'
    // codes share lines of 128 bytes.
    const int id = static_cast<int>(blockIdx.x), turn = id / 8, upper = turn / a.by_kv_heads, g = turn - upper * p.kv_heads;
    const int unit = upper * 8 + id % 8;
    if (unit >= args.units) return;
    const int group = p.heads / p.kv_heads;
    Kv4Unit u{};
    u.splits = 1;
    if (!(a.parts > 0 ? dealtUnit<ROWS>(p, group, unit, args.units, a.parts, u) : rowBlock<ROWS>(p, group, unit, u.s, u.r0))) return;
    const SeqSpan s{uniform(u.s.q0), uniform(u.s.k0), static_cast<int32_t>(uniform(u.s.nq)), static_cast<int32_t>(uniform(u.s.nk))};
    const int r0 = __builtin_amdgcn_readfirstlane(u.r0), split = __builtin_amdgcn_readfirstlane(u.split), splits = __builtin_amdgcn_readfirstlane(u.splits);
    const int rows = s.nq * group;
    // Keys that a row sees: those below its limit.
    auto limit = [&](int r) {
        return p.causal != 0 ? min(max(min(r, rows - 1) / a.by_group + s.nk - s.nq + 1, 0), s.nk) : s.nk;
    };
    const int limLo = __builtin_amdgcn_readfirstlane(limit(r0)), limHi = __builtin_amdgcn_readfirstlane(limit(r0 + ROWS - 1));
    int lim[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) lim[b] = limit(r0 + b * EDGE + col) - 4 * part;
    const int tiles = (limHi + 31) / 32, each = __builtin_amdgcn_readfirstlane(tiles / splits), more = tiles - each * splits;
    const int first = each * split + min(split, more) + wave;
    const int end = each * split + min(split, more) + each + (split < more ? 1 : 0);
    const int token0 = __builtin_amdgcn_readfirstlane(r0 / a.by_group);
    auto tokenOf = [&](int r) { return r / a.by_group - token0; };
    auto headOf = [&](int r, int t) { return r - (t + token0) * group + g * group; };

    // Where sixteen elements of a head lie in LDS, from which on (-1: nowhere). A
    // head of half a piece more than whole ones has its last 16 bytes as a piece,
    // the first eight of them a second time.
    const int bytes = p.dim / 2, lastPiece = (bytes - 1) / 16;
    const bool half = bytes % 16 != 0;
    auto elementsAt = [&](int unit16) {
        const int n = half && unit16 >= 2 * lastPiece ? (unit16 == 2 * lastPiece + 1 ? 2 * lastPiece : -1) : unit16;
        return n >= 0 && n * 16 < p.dim ? n * 16 : -1;
    };

    // This wave's loads of a tile: row and piece of each, by lane.
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ldsTiles)) + wave * S::kRing;
    const char *const k0 = static_cast<const char*>(p.k) + s.k0 * p.k_stride + static_cast<int64_t>(g) * bytes,
               *const v0 = static_cast<const char*>(p.v) + s.k0 * p.v_stride + static_cast<int64_t>(g) * bytes;
    // Rows of a tile lie less than 2^24 bytes apart, keys of 31 of them and scales too.
    const uint32_t ks = static_cast<uint32_t>(p.k_stride), vs = static_cast<uint32_t>(p.v_stride), heads4 = p.kv_heads * 4;
    const char* const scales = reinterpret_cast<const char*>((ln < 32 ? args.k_scale : args.v_scale) + s.k0 * p.kv_heads + g);
    uint32_t place = lds0;   // of the next tile to ask for
    auto load = [&](int it) __attribute__((always_inline)) {
        const int64_t j0 = static_cast<int64_t>(it) * 32;
        const int last = limHi - 1 - it * 32;   // keys behind the last repeat it
        const char *const kt = reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(k0 + j0 * p.k_stride))),
                   *const vt = reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(v0 + j0 * p.v_stride)));
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const int row = (i * 64 + ln) / S::kPieces, piece = ln % S::kPieces ^ S::swizzle(row);
            const uint32_t at = piece == lastPiece ? bytes - 16 : piece * 16, j = min(row, last);
            if (piece <= lastPiece) {
                S::dma16(kt, __umul24(j, ks) + at, place + i * 1024);
                S::dma16(vt, __umul24(j, vs) + at, place + S::kHalf + i * 1024);
            }
        }
        S::dma4(scales + j0 * heads4 + __umul24(min(ln & 31, last), heads4), place + 2 * S::kHalf);
        place = place == lds0 + (S::kStages - 1) * S::kStage ? lds0 : place + S::kStage;
    };
#pragma unroll
    for (int n = 0; n < S::kStages - 1; ++n) {
        if (first + n * NW < end) load(first + n * NW);
    }

    // Queries: step i takes the eight elements whose codes a lane's i-th word holds.
    Piece<Q> q[S::kPartsQ][QB][KS];
    using V8 = T __attribute__((ext_vector_type(8)));
    auto queries = [&](int b, auto take) __attribute__((always_inline)) {
        const int r = min(r0 + b * EDGE + col, rows - 1), t = tokenOf(r);
        const T* row = static_cast<const T*>(p.q) + (s.q0 + token0 + t) * p.q_stride + static_cast<int64_t>(headOf(r, t)) * p.dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int place = part * KS + i, d = elementsAt(place / 2);
            V8 v = {};
            if (d >= 0) v = *reinterpret_cast<const V8*>(row + d + place % 2 * 8);
            take(i, v);
        }
    };
    auto hold = [&](int b, int i, V8 v) __attribute__((always_inline)) {
        if constexpr (S::kPartsQ == 1) {
            q[0][b][i] = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float left = v[e];
#pragma unroll
                for (int n = 0; n < S::kPartsQ; ++n) {
                    q[n][b][i][e] = static_cast<Q>(left);
                    left -= static_cast<float>(q[n][b][i][e]);
                }
            }
        }
    };
    static_assert(QB == 1, "c is of a lane's one query");
    float c = args.c;
    Sizes<T> sizes;
    queries(0, [&](int i, V8 v) {
        sizes.take(v);
        hold(0, i, v);
    });
    // Queries far from one are taken times a power of two, a row's all alike, and their
    // scores' c times its reciprocal: c is a lane's own, so that tiles are as they were
    // (a token over 100 keys 4.96 us for 4.84, prompts 1 % more).
    if (__builtin_expect(args.up != 0 || __any(sizes.far()), 0)) {
        float top = 0.0f;
        queries(0, [&](int, V8 v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(static_cast<float>(v[e])));
        });
        top = largestOf<EDGE>(top);
        const int size = __builtin_amdgcn_frexp_expf(top);
        const bool some = top > 0.0f && top < INFINITY;
        const int by = some ? min(max(args.up, S::kLeast - size), S::kMost - size) : args.up;
        queries(0, [&](int i, V8 v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(__builtin_amdgcn_ldexpf(static_cast<float>(v[e]), by));
            hold(0, i, v);
        });
        c = __builtin_amdgcn_ldexpf(c, args.up - by);
    }
    // They are taken here: the compiler knows nothing of the loads to LDS and would
    // wait for these, and so for all, in every tile.
#pragma unroll
    for (int n = 0; n < S::kPartsQ; ++n) {
#pragma unroll
        for (int b = 0; b < QB; ++b) {
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                i32x4 bits = __builtin_bit_cast(i32x4, q[n][b][i]);
                asm volatile("" : "+v"(bits));
                q[n][b][i] = __builtin_bit_cast(Piece<Q>, bits);
            }
        }
    }

    // A lane's words of key block kb: those of row kb EDGE + col from `part` on.
    constexpr int WB = KS * 4;   // bytes of them
    auto words = [&](const char* tile, int kb, int (&w)[KS]) __attribute__((always_inline)) {
        const int row = kb * EDGE + col, turned = S::swizzle(row) << 4;
        constexpr int READ = WB % 16 == 0 ? 16 : WB % 8 == 0 ? 8 : 4;
        using Words = int __attribute__((ext_vector_type(READ / 4)));
#pragma unroll
        for (int i = 0; i < KS; i += READ / 4) {
            const int byte = part * WB + i * 4;
            const auto v = *reinterpret_cast<const Words*>(tile + row * S::kPitch + (byte ^ turned));
            if constexpr (READ == 4) {
                w[i] = v[0];
            } else {
#pragma unroll
                for (int e = 0; e < READ / 4; ++e) w[i + e] = v[e];
            }
        }
    };
    // The row whose eight bytes this lane hands the transposing read, and where.
    const int j16 = ln & 15;
    const int vrow = EDGE == 32 ? 8 * (j16 >> 2) + 4 * part + (j16 & 3) : 16 * ((j16 >> 2) & 1) + 4 * part + (j16 & 3);
    const uint32_t vat = vrow * S::kPitch + (S::swizzle(vrow) << 4) + (EDGE == 32 ? (ln >> 4) & 1 : j16 >> 3) * 8;

    F32<NO> o[QB][DB] = {};
    float m[QB], l[QB];   // what the weights of this lane's queries are relative to; of this lane's keys, their sum
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        m[b] = kLowest;
        l[b] = 0.0f;
    }
    constexpr int kApart = EDGE == 32 ? 8 : 16;   // between the fours of keys that a lane holds
    int taken = 0;   // the tile's place
    for (int it = first; it < end; it += NW) {
        const char* const tile = ldsTiles + wave * S::kRing + taken;
        taken = taken == (S::kStages - 1) * S::kStage ? 0 : taken + S::kStage;
        S::wait(it + NW < end ? 1 : 0);
        // Into the place of the tile before, whose values are in their sums.
        if (it + (S::kStages - 1) * NW < end) load(it + (S::kStages - 1) * NW);
        F32<NO> x[QB][KB] = {};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            int w[KS];
            words(tile, kb, w);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const Piece<Q> k = numbers<Q>(w[i], args.codes);
#pragma unroll
                for (int b = 0; b < QB; ++b) {
#pragma unroll
                    for (int n = 0; n < S::kPartsQ; ++n) x[b][kb] = product<EDGE>(k, q[n][b][i], x[b][kb]);
                }
            }
        }
        f32x4 kScale[NS / 4], vScale[NS / 4];
#pragma unroll
        for (int e = 0; e < NS / 4; ++e) {
            const float* const at = reinterpret_cast<const float*>(tile + 2 * S::kHalf) + kApart * e + 4 * part;
            kScale[e] = *reinterpret_cast<const f32x4*>(at) * c;
            vScale[e] = *reinterpret_cast<const f32x4*>(at + 32);
        }
        const bool edge = limLo < it * 32 + 32;
        Piece<__bf16> w[QB][S::kPartsW][NS / 8];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int seen = lim[b] - it * 32;   // keys of this lane's, counted as the scores are
            float y[NS];
#pragma unroll
            for (int e = 0; e < NS; ++e) y[e] = x[b][e / NO][e % NO] * kScale[e / 4][e % 4];
            if (edge) {
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    y[e] = kApart * (e / 4) + e % 4 < seen ? y[e] : -INFINITY;
                    asm volatile("" : "+v"(y[e]));   // a branch
                }
            }
            float top = y[0];
#pragma unroll
            for (int e = 1; e < NS; ++e) top = fmaxf(top, y[e]);
            top = largestOf<EDGE>(top);
            if (__any(top > m[b] + 8.0f)) {
                const float base = fmaxf(m[b], top), keep = __builtin_amdgcn_exp2f(m[b] - base);
                m[b] = base;
                l[b] *= keep;
#pragma unroll
                for (int i = 0; i < DB; ++i) {
#pragma unroll
                    for (int e = 0; e < NO; ++e) o[b][i][e] *= keep;
                }
            }
#pragma unroll
            for (int e = 0; e < NS; ++e) {
                y[e] = __builtin_amdgcn_exp2f(y[e] - m[b]);
                l[b] += y[e];
                y[e] *= vScale[e / 4][e % 4];
            }
            if (edge) {   // a hidden value's scale may be anything
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    y[e] = kApart * (e / 4) + e % 4 < seen ? y[e] : 0.0f;
                    asm volatile("" : "+v"(y[e]));
                }
            }
#pragma unroll
            for (int e = 0; e < NS; ++e) {
                float left = y[e];
#pragma unroll
                for (int n = 0; n < S::kPartsW; ++n) {
                    w[b][n][e / 8][e % 8] = static_cast<__bf16>(left);
                    left -= static_cast<float>(w[b][n][e / 8][e % 8]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < DT / 32; ++i) {
            using Lds = __attribute__((address_space(3))) i32x2;
            const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32((Lds*)(tile + S::kHalf + (vat ^ (i << 4))));
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                // Of 32 columns a read's halves are those of the first and the second
                // eight keys, of 16 those of two blocks of columns.
                const Piece<__bf16> vv = numbers<__bf16>(v[n], 1.0f);
                const int block = EDGE == 32 ? i : 2 * i + n, keys = EDGE == 32 ? n : 0;
#pragma unroll
                for (int b = 0; b < QB; ++b) {
#pragma unroll
                    for (int k = 0; k < S::kPartsW; ++k) o[b][block] = product<EDGE>(vv, w[b][k][keys], o[b][block]);
                }
            }
        }
    }

    // The waves' sums by rows through LDS, 16 rows at a time and 16 bytes a lane,
    // joined on the way out.
    char* const sums = ldsTiles;
    float2* const tops = reinterpret_cast<float2*>(ldsTiles + NW * 16 * S::kRow);
    constexpr int LPR = DT <= 64 ? 16 : DT <= 128 ? 32 : 64, SIDE = 64 / LPR;   // lanes of a row, rows side by side
    const int piece = ln % LPR, d0 = piece * 4 < DT ? elementsAt(piece / 4) : -1, d = d0 + piece % 4 * 4;
    auto meet = [] {
        if constexpr (NW > 1) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    };
#pragma unroll
    for (int b = 0; b < QB; ++b) l[b] = sumOf<EDGE>(l[b]);
#pragma unroll
    for (int row0 = 0; row0 < ROWS; row0 += 16) {
        if (r0 + row0 >= rows) break;
        meet();   // all are done with what lay there
        constexpr int kBlocks = EDGE == 16 ? 16 : 32;
        const int b = row0 / kBlocks;
        const int row = EDGE == 16 ? col : b * 32 + col - row0;   // of the sixteen
        if (row >= 0 && row < 16 && r0 + row0 + row < rows) {
            char* const at = sums + (wave * 16 + row) * S::kRow;
#pragma unroll
            for (int i = 0; i < DB; ++i) {
#pragma unroll
                for (int e = 0; e < NO; e += 4) {
                    const int to = (i * EDGE + (EDGE == 32 ? 8 * (e / 4) : 0)) / 4 + part;
                    *reinterpret_cast<f32x4*>(at + ((to ^ (row & 7)) << 4)) = f32x4{o[b][i][e], o[b][i][e + 1], o[b][i][e + 2], o[b][i][e + 3]};
                }
            }
            if (part == 0) tops[wave * 16 + row] = make_float2(m[b], l[b]);
        }
        meet();
        for (int at16 = wave * SIDE + ln / LPR; at16 < min(16, rows - r0 - row0); at16 += NW * SIDE) {
            float2 ml[NW];
            float top = kLowest, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                ml[w] = tops[w * 16 + at16];
                top = fmaxf(top, ml[w].x);
            }
            f32x4 v = {};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float keep = NW == 1 ? 1.0f : __builtin_amdgcn_exp2f(ml[w].x - top);
                sum += ml[w].y * keep;
                if (d0 >= 0) v += *reinterpret_cast<const f32x4*>(sums + (w * 16 + at16) * S::kRow + ((piece ^ (at16 & 7)) << 4)) * keep;
            }
            const int r = r0 + row0 + at16, t = tokenOf(r), h = headOf(r, t);
            const int64_t at = (s.q0 + token0 + t) * p.heads + h;
            if (a.parts > 0 && split == 0) {   // ranges that this row does not have
                for (int n = splits + piece; n < a.parts; n += LPR) a.ml[static_cast<int64_t>(n) * p.q_rows * p.heads + at] = make_float2(kLowest, 0.0f);
            }
            if (piece == 0) {
                if (a.parts > 0) a.ml[static_cast<int64_t>(split) * p.q_rows * p.heads + at] = make_float2(top, sum);
                else if (p.lse != nullptr) p.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
            }
            if (d0 < 0) continue;
            if (a.parts > 0) {
                *reinterpret_cast<f32x4*>(a.acc + (static_cast<int64_t>(split) * p.q_rows * p.heads + at) * p.dim + d) = v;
            } else {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                Vec4<T> out;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(v[e] * inv);
                *reinterpret_cast<Vec4<T>*>(static_cast<T*>(p.out) + (s.q0 + token0 + t) * p.out_stride + static_cast<int64_t>(h) * p.dim + d) = out;
            }
        }
    }
}

}  // namespace mlk
