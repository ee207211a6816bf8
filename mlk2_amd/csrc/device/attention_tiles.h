// Attention on matrix cores: NW waves, 32 query rows each, over tiles of keys
// in LDS, for rows whose heads are whole 16-byte pieces.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "attention_span.h"

namespace mlk {

using f32x16 = float __attribute__((ext_vector_type(16)));
using f32x4 = float __attribute__((ext_vector_type(4)));
template <typename T>
using Vec4 = T __attribute__((ext_vector_type(4)));
/// 16 bytes of a row.
template <typename T>
using Piece = T __attribute__((ext_vector_type(16 / sizeof(T))));

constexpr float kLowest = -3.402823466e38f;   // a running maximum before any score
constexpr float kFar = 16777216.0f;           // 2^24

/// c += a b over the columns of a piece in either half wave: 16 of f16 and
/// bf16, 8 of f32.
__device__ __forceinline__ f32x16 mfma(Piece<_Float16> a, Piece<_Float16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Piece<__bf16> a, Piece<__bf16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Piece<float> a, Piece<float> b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

/// The other half wave's value of the same query (lanes l and l ^ 32).
__device__ __forceinline__ float otherHalf(float v) {
    const int i = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) != 0 ? r[0] : r[1]);
}

/// Orders a block of NV products of two LDS reads each and NK of one each:
/// every product's reads AHEAD products before it.
template <int NV, int NK, int AHEAD, int J = -1>
__device__ __forceinline__ void readAhead() {
    constexpr int reads = J >= 0 ? (J + AHEAD < NV ? 2 : J + AHEAD < NV + NK ? 1 : 0)
                          : AHEAD <= NV ? 2 * AHEAD : NV + (AHEAD < NV + NK ? AHEAD : NV + NK);
    if constexpr (J >= 0) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (reads > 0) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
    if constexpr (J + 1 < NV + NK) readAhead<NV, NK, AHEAD, J + 1>();
}

/// n / d for n < 2^30 by a product: mul = ceil(2^(31 + L) / d), 2^L the power
/// of two at or above d, is off d's reciprocal by less than 2^L / 2^(31 + L).
struct Divider {
    uint32_t mul;   // 0: d is 1
    int shift;      // L - 1
};
__device__ __forceinline__ int operator/(int n, const Divider& d) {
    return d.mul == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), d.mul) >> d.shift);
}

/// What a launch of tiles works on: which keys, which rows, and where the
/// results go.
struct TileArgs {
    mlkd_attention p;
    int keys;         // 1: the prefix, 2: the sequences' own, 3: both
    int all_rows;     // 1: the rows that sequences hold, all together (prefix keys only)
    int splits;       // key ranges of each row block
    int part0;        // partial results: the first range's index ...
    int parts;        // ... of so many (0: results go straight to out)
    float* acc;       // [parts][rows * heads][dim]
    float2* ml;       // [parts][rows * heads]: maximum (times log2 e), sum
    Divider by_group, by_kv_heads, by_splits, by_heads;
};

/// A value that all lanes have alike, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
    return static_cast<int64_t>(hi) << 32 | lo;
}

__device__ __forceinline__ int64_t laneOf(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<int64_t>(hi) << 32 | lo;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int addFrom(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}

/// The sum of the lanes up to and with this one.
__device__ __forceinline__ int sumUpTo(int v) {
    v = addFrom<0x111, 0xf>(v);   // rows of 16 lanes, from 1, 2, 4, 8 before
    v = addFrom<0x112, 0xf>(v);
    v = addFrom<0x114, 0xf>(v);
    v = addFrom<0x118, 0xf>(v);
    v = addFrom<0x142, 0xa>(v);   // the last lane of rows 0 and 2 to rows 1 and 3
    return addFrom<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
}

/// The row block `tile` counted from the end of the batch: its sequence and
/// first row. Rows are (token, head of the group); each sequence has
/// ceil(nq * group / ROWS) blocks. A lane reads a sequence's lengths. All lanes
/// return the same; false past the first block.
template <int ROWS>
__device__ __forceinline__ bool rowBlock(const mlkd_attention& p, int group, int tile, SeqSpan& s, int& r0) {
    const int ln = threadIdx.x & 63;
    for (int s0 = p.sequences - 1; s0 >= 0; s0 -= 64) {
        SeqSpan of{};
        if (s0 >= ln) of = spanOf(p, s0 - ln);
        const int sum = sumUpTo((of.nq * group + ROWS - 1) / ROWS);
        const uint64_t past = __ballot(sum > tile);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            s = SeqSpan{laneOf(of.q0, at), laneOf(of.k0, at), __builtin_amdgcn_readlane(of.nq, at), __builtin_amdgcn_readlane(of.nk, at)};
            r0 = (__builtin_amdgcn_readlane(sum, at) - 1 - tile) * ROWS;
            return true;
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

/// Keys (or values) in LDS: rows of RB bytes in 16-byte pieces, piece c of row
/// j at c ^ swizzle(j), so that the reads below meet every bank once: keys are
/// read 16 rows x 16 bytes at a time, 16-bit values 4 rows x 64 bytes, f32 values
/// two rows four apart x 128 bytes.
template <int RB>
__device__ __forceinline__ int swizzleK(int j) {
    return RB == 128 ? (j >> 1) & 7 : j & 15;
}
template <typename T, int RB>
__device__ __forceinline__ int swizzleV(int j) {
    return sizeof(T) == 4 ? (j >> 2 & 1) << 3 : RB == 128 ? (j >> 1 & 1) << 2 : (j & 3) << 2;
}

/// NW waves of 32 rows each, in KG groups: those of a group have different
/// rows, the groups the same rows and different keys of a tile. Their sums are
/// joined at the end.
template <typename T, int DT, int NW, int KG, int KEYS, int STAGES>
struct Tiles {
    static constexpr int KS = DT * sizeof(T) / 32, DB = DT / 32;      // steps of q k^T, two pieces each; 32-column blocks of out
    static constexpr int RB = (DT <= 64 ? 64 : DT <= 128 ? 128 : 256) * sizeof(T);
    static constexpr int kTile = KEYS * RB;                          // bytes of a tile of keys
    static constexpr int kStage = 2 * kTile;
    static constexpr int kLds = STAGES * kStage;
    static constexpr int kRows = 32 * NW / KG;
    static constexpr int IPW = kTile / 1024 / NW;                    // 1024-byte loads of a wave, for keys and again for values
    static constexpr int kKeys = KEYS / KG, KB = kKeys / 32;         // keys of a tile that a wave takes
    /// log2 of a largest weight when the weights' reference is set: see attentionTiles.
    static constexpr float kTop = std::is_same_v<T, _Float16> ? 7.0f : 0.0f;
    static_assert(IPW >= 1 && IPW * NW * 1024 == kTile, "a tile is whole loads of the waves");
    static_assert(STAGES == 2 || (STAGES - 2) * 2 * IPW <= 63, "the loads waited on by number fit the counter");

    /// 16 bytes a lane to LDS at `m0` + 16 * lane. A load to LDS takes M0 one
    /// wait state after a scalar write of it at the earliest; the compiler puts
    /// none inside asm (s_nop 0).
    static __device__ __forceinline__ void dma(const void* base, uint32_t off, uint32_t m0) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
    }

    static __device__ __forceinline__ int swizzle(int half, int row) {
        return half == 0 ? swizzleK<RB>(row) : swizzleV<T, RB>(row);
    }

    /// This wave's loads of a tile's keys (half 0) or values (1), straight to
    /// LDS: rows past the last valid one repeat it; pieces past the head dim
    /// stay zero.
    static __device__ __forceinline__ void load(int half, const char* from, uint32_t stride, int last, int pieces, uint32_t lds, int wave) {
        constexpr int P = RB / 16, R = 64 / P;   // pieces of a row, rows of a load
        from = reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(from)));
        int ln = threadIdx.x & 63;
        asm volatile("" : "+v"(ln));   // the offsets are taken anew for each tile: kept, they are up to 64 registers
        if (last >= KEYS - 1 && pieces == P) {
            const int w0 = wave * IPW * R;
            const uint32_t row = ln / P * stride, piece = ((ln % P) ^ swizzle(half, w0 + ln / P)) << 4;
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                // Rows i R + r with r < R: their swizzle is i R's and r's.
                const int turned = swizzle(half, w0 + i * R) ^ swizzle(half, w0);
                dma(from + static_cast<uint64_t>(w0 + i * R) * stride, (piece ^ (turned << 4)) + row, lds + half * kTile + (wave * IPW + i) * 1024);
            }
            return;
        }
#pragma unroll 1
        for (int i = 0; i < IPW; ++i) {
            const int n = wave * IPW + i, row = n * R + ln / P, piece = (ln % P) ^ swizzle(half, row);
            const uint32_t off = static_cast<uint32_t>(min(row, last)) * stride + piece * 16;
            if (piece < pieces) dma(from, off, lds + half * kTile + n * 1024);
        }
    }

    /// Waits until at most `ahead` tiles of this wave's loads are in flight.
    static __device__ __forceinline__ void wait(int ahead) {
        static_assert(STAGES <= 4, "");
        if (ahead >= 2 && STAGES >= 4) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * 2 * IPW) : "memory");
        else if (ahead >= 1 && STAGES >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * IPW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};

/// One row block of one key/value head. With S^T = K Q^T in 32 x 32 blocks a
/// lane holds 16 keys' scores of one query (the other 16 in lane ^ 32), so the
/// softmax is register work but for one exchange of maxima, and its weights are
/// as they stand the operand of out^T = V^T W^T: the keys of a 16-key step are
/// taken in the order the scores have. V^T comes out of V's rows in LDS by
/// transposing reads. The maximum that the weights are taken relative to
/// follows the running one only when that has grown by 2^8: sums of weights
/// up to 2^8 lose nothing in f32, and out is rescaled in few tiles. Weights are
/// rounded to the type as the product's operand, half a step, relative, their
/// sum is of the f32 values. f16 has such steps from 2^-14 on and 0 below 2^-25:
/// its weights are 2^7 to 2^15 at the row's maximum instead of 1 to 2^8, so that
/// only weights below 2^-32 of the largest, not 2^-25, are in the sum alone.
///
/// What bounds it: 16-bit types of 128 columns, the products (a wave's 32 of a
/// 64-key tile take 1024 cycles and more with the LDS reads that feed them)
/// and the weights (950, 32 exponentials a lane) about equally; of 64 columns
/// the weights; f32 the products; single tokens the reads of keys and values.
/// Eight waves share a tile, so that it is read from L2 once for 256 rows, and
/// take turns (all in step, the 8 prompts below took 666 us). Two workgroups of
/// 64 columns fit a compute unit at 128 registers (16 sequences of up to 1024,
/// 16 heads: 78 -> 64 us).
/// Measured (bf16, 32 and 8 heads of 128, causal): 8 packed prompts of up to
/// 4096 tokens 546 us, 945 TFLOP/s; one of 2048, by halves, 56 us, 610
/// TFLOP/s; 32 single tokens over up to 8192 keys 148 us, 4.2 TB/s. f32, two
/// sequences of 1001, 8 heads of 64: 46 us.
template <typename T, int DT, int NW, int KG, int KEYS, int STAGES>
__global__ __launch_bounds__(NW * 64, DT > 128 ? 1 : DT == 64 && sizeof(T) == 2 ? 4 : 2) void attentionTiles(TileArgs a) {
    using S = Tiles<T, DT, NW, KG, KEYS, STAGES>;
    using P = Piece<T>;
    using V4 = Vec4<T>;
    using Short4 = short __attribute__((ext_vector_type(4)));
    constexpr int KS = S::KS, DB = S::DB, RB = S::RB, KB = S::KB;
    constexpr bool PING = NW == 8;
    extern __shared__ __align__(16) char ldsTiles[];
    const mlkd_attention& p = a.p;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int ln = threadIdx.x & 63, l32 = ln & 31, hl = ln >> 5;
    const int id = static_cast<int>(blockIdx.x), of = id / a.by_kv_heads, g = id - of * p.kv_heads;
    const int rest = of / a.by_splits, split = of - rest * a.splits, group = p.heads / p.kv_heads;
    int np = (a.keys & 1) != 0 ? prefixOf(p) : 0;
    SeqSpan s{};
    int r0 = rest * S::kRows;
    if (a.all_rows != 0) {
        s = heldRows(p);
        if (r0 >= s.nq * group) return;
    } else if (!rowBlock<S::kRows>(p, group, rest, s, r0)) {
        return;
    }
    s = SeqSpan{uniform(s.q0), uniform(s.k0), static_cast<int32_t>(uniform(s.nq)), static_cast<int32_t>(uniform(s.nk))};
    r0 = __builtin_amdgcn_readfirstlane(r0);
    np = __builtin_amdgcn_readfirstlane(np);
    const int rows = s.nq * group;
    // Keys that a row sees: the prefix, and own keys below lim = token + slope.
    const int nk = (a.keys & 2) != 0 ? s.nk : 0;
    auto limit = [&](int r) {
        return p.causal != 0 ? min(max(min(r, rows - 1) / a.by_group + s.nk - s.nq + 1, 0), nk) : nk;
    };
    const int tilesP = (np + KEYS - 1) / KEYS, tiles = tilesP + (limit(r0 + S::kRows - 1) + KEYS - 1) / KEYS;
    // Tiles of this range: so many each, the first `more` one more.
    const int each = tiles / a.by_splits, more = tiles - each * a.splits;
    const int first = __builtin_amdgcn_readfirstlane(each * split + min(split, more));
    const int end = __builtin_amdgcn_readfirstlane(first + each + (split < more ? 1 : 0));
    const int rw = r0 + wave % (NW / KG) * 32, key0 = wave / (NW / KG) * S::kKeys;   // this wave's first row, first key of a tile
    const int limLo = limit(rw), limHi = limit(rw + 31);
    const int lim = limit(rw + l32);
    // Row r of the block's sequence: its token, counted from the block's first,
    // and its elements' place, counted from that token's.
    const int token0 = __builtin_amdgcn_readfirstlane(r0 / a.by_group);
    auto tokenOf = [&](int r) { return r / a.by_group - token0; };
    auto placeOf = [&](int r, int64_t stride) {
        const int t = tokenOf(r);
        return static_cast<uint32_t>(t) * static_cast<uint32_t>(stride) + static_cast<uint32_t>((r - (t + token0) * group + g * group) * p.dim);
    };

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ldsTiles));
    const int pieces = p.dim * static_cast<int>(sizeof(T)) / 16;
    if (p.dim < DT) {   // what the loads leave out
        for (int i = threadIdx.x * 16; i < S::kLds; i += NW * 64 * 16) *reinterpret_cast<f32x4*>(ldsTiles + i) = f32x4{};
        __syncthreads();
    }
    // Queries, a piece a step; a negative scale turns their signs. Eight waves
    // ask for them by whole rows, to the LDS of the last two stages: the 16
    // bytes of 64 rows that a step takes are 64 cycles of a load otherwise, 16
    // loads a wave.
    const float c = static_cast<float>(fabs(p.scale) * 1.4426950408889634);
    constexpr int kPieces = RB / 16, kRowsOfLoad = 64 / kPieces;
    const T* q0 = static_cast<const T*>(p.q) + (s.q0 + token0) * p.q_stride;
    static_assert(!PING || NW * 32 * RB == 2 * S::kStage, "the queries take the last two stages");
    constexpr int kQueries = 2 * S::kStage / NW;   // of a wave
    const uint32_t atQ = S::kLds - 2 * S::kStage + wave * kQueries;
    P q[KS];
    auto askQueries = [&] {
        if constexpr (PING) {
#pragma unroll
            for (int i = 0; i < 32 / kRowsOfLoad; ++i) {
                const int row = i * kRowsOfLoad + ln / kPieces, piece = (ln % kPieces) ^ swizzleK<RB>(row);
                const uint32_t off = placeOf(min(rw + row, rows - 1), p.q_stride) * static_cast<uint32_t>(sizeof(T)) + piece * 16;
                if (piece < pieces) S::dma(q0, off, lds0 + atQ + i * 1024);
            }
        } else {
            const T* row = q0 + placeOf(min(rw + l32, rows - 1), p.q_stride);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int d = (2 * i + hl) * (16 / static_cast<int>(sizeof(T)));
                q[i] = P{};
                if (d < p.dim) q[i] = *reinterpret_cast<const P*>(row + d);
            }
        }
    };
    auto takeQueries = [&] {
        if constexpr (PING) {
            const char* at = ldsTiles + atQ;
#pragma unroll
            for (int i = 0; i < KS; ++i) q[i] = *reinterpret_cast<const P*>(at + l32 * RB + (((2 * i + hl) ^ swizzleK<RB>(l32)) << 4));
        }
        if (p.scale < 0.0) {
#pragma unroll
            for (int i = 0; i < KS; ++i) q[i] = -q[i];
        }
    };
    // The next tile to load: its rows, how many of its keys are left, its place.
    struct Next {
        const char *k, *v;
        uint32_t ks, vs;   // bytes from row to row
        int left, at;
    };
    auto rowsFrom = [&](const void* k, const void* v, int64_t ks, int64_t vs, int64_t row, int left) {
        constexpr int64_t size = sizeof(T);
        return Next{static_cast<const char*>(k) + (row * ks + static_cast<int64_t>(g) * p.dim) * size,
                    static_cast<const char*>(v) + (row * vs + static_cast<int64_t>(g) * p.dim) * size,
                    static_cast<uint32_t>(ks * size), static_cast<uint32_t>(vs * size), left, 0};
    };
    auto start = [&](int it) {
        const int64_t j = static_cast<int64_t>(it < tilesP ? it : it - tilesP) * KEYS;
        return it < tilesP ? rowsFrom(p.prefix_k, p.prefix_v, p.prefix_k_stride, p.prefix_v_stride, j, np - static_cast<int>(j))
                           : rowsFrom(p.k, p.v, p.k_stride, p.v_stride, s.k0 + j, nk - static_cast<int>(j));
    };
    Next next = start(first);
    auto load = [&](int it) {
        if (it == tilesP && it > first) {   // from the prefix to the sequence's own keys
            const int at = next.at;
            next = start(it);
            next.at = at;
        }
        S::load(0, next.k, next.ks, next.left - 1, pieces, lds0 + next.at, wave);
        S::load(1, next.v, next.vs, next.left - 1, pieces, lds0 + next.at, wave);
        next.k += static_cast<uint64_t>(KEYS) * next.ks;
        next.v += static_cast<uint64_t>(KEYS) * next.vs;
        next.left -= KEYS;
        next.at = next.at == (STAGES - 1) * S::kStage ? 0 : next.at + S::kStage;
    };

    // Offsets of this lane's reads within a tile.
    const uint32_t atK = l32 * RB + ((hl ^ swizzleK<RB>(l32)) << 4);   // step i: its piece bits turned by 2 i
    uint32_t atV[DB];
    // 16-bit values: the row of four, and their eight bytes, that this lane
    // hands the transposing read; f32: the first row and its column.
    const int vr = 4 * hl + (sizeof(T) == 4 ? 0 : (ln & 15) / 4);
#pragma unroll
    for (int i = 0; i < DB; ++i) {
        const int byte = sizeof(T) == 4 ? i * 128 + l32 * 4 : i * 64 + ((ln >> 4) & 1) * 32 + (ln & 3) * 8;
        atV[i] = S::kTile + vr * RB + (((byte >> 4) ^ swizzleV<T, RB>(vr)) << 4) + (byte & 15);
    }

    f32x16 o[DB] = {};
    float m = kLowest, l = 0.0f;   // what the weights of this lane's query are relative to; of this lane's keys, their sum
    auto place = [&](int it) { return ldsTiles + (it - first) % STAGES * S::kStage + key0 * RB; };
    auto firstKey = [&](int it) { return (it < tilesP ? it : it - tilesP) * KEYS + key0; };
    // Scores of a tile.
    f32x16 x[KB];
    auto scores = [&](int it) {
        const char* tile = place(it);
        uint32_t lane = atK;
        if (KS > 8) asm volatile("" : "+v"(lane));   // taken anew for each tile, where 16 of them take registers
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) x[kb] = f32x16{};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) x[kb] = mfma(*reinterpret_cast<const P*>(tile + kb * 32 * RB + (lane ^ (i << 5))), q[i], x[kb]);
        }
    };
    // Their weights, in place for f32, else rounded to the type.
    P w[sizeof(T) == 4 ? 1 : S::kKeys / 16];
    auto weights = [&](int it) {
        const int j0 = firstKey(it);
        if ((it < tilesP ? np : limLo) < j0 + S::kKeys) {
            const int seen = (it < tilesP ? np : lim) - j0 - 4 * hl;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[kb][e] = kb * 32 + 8 * (e / 4) + e % 4 < seen ? x[kb][e] : -INFINITY;
                asm volatile("" : "+v"(x[kb]));   // a branch: selects would cost every tile a hundred instructions
            }
        }
        float top = x[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, x[kb][e]);
        }
        top = __builtin_fmaf(fmaxf(top, otherHalf(top)), c, -S::kTop);
        while (__any(top > m + 8.0f)) {   // once at most; as an if it has out copied in every tile
            const float base = fmaxf(m, top), keep = __builtin_amdgcn_exp2f(m - base);
            m = base;
            l *= keep;
#pragma unroll
            for (int i = 0; i < DB; ++i) {
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= keep;
            }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][e], c, -m));
                l += v;
                if constexpr (sizeof(T) == 4) x[kb][e] = v;
                else w[kb * 2 + e / 8][e % 8] = static_cast<T>(v);
            }
        }
        // They are taken here: the compiler would move them behind the barrier, to their use.
        asm volatile("" : "+v"(l));
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) asm volatile("" : "+v"(x[kb]));
        } else {
#pragma unroll
            for (int kg = 0; kg < S::kKeys / 16; ++kg) {
                f32x4 bits = __builtin_bit_cast(f32x4, w[kg]);
                asm volatile("" : "+v"(bits));
                w[kg] = __builtin_bit_cast(P, bits);
            }
        }
    };
    // The weights' sums of values.
    auto values = [&](int it) {
        const char* tile = place(it);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
#pragma unroll
                    for (int i = 0; i < DB; ++i) {
                        const float v = *reinterpret_cast<const float*>(tile + atV[i] + (kb * 32 + 8 * (e / 4) + e % 4) * RB);
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, x[kb][e], o[i], 0, 0, 0);
                    }
                }
            }
        } else {
#pragma unroll
            for (int kg = 0; kg < S::kKeys / 16; ++kg) {
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    using Lds = __attribute__((address_space(3))) Short4;
                    const char* at = tile + atV[i] + kg * 16 * RB;
                    const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(at));
                    const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(at + 8 * RB));
                    const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[i] = mfma(__builtin_bit_cast(P, both), w[kg], o[i]);
                }
            }
        }
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        if (NW > 1) __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    const int mine = min(end, tilesP + (limHi + KEYS - 1) / KEYS);   // this wave's last tile, and one
    // A tile takes two phases: its weights on the vector units, then its values
    // and the next tile's scores on the matrix cores. Of eight waves, two on
    // each SIMD, the second four run half a tile late: while one wave of a SIMD
    // is in one phase, the other is in the other.
    const bool late = PING && wave >= NW / 2;
    if constexpr (STAGES == 2) {   // no room to have the next tile's keys early
        if (first < end) {
            askQueries();
            takeQueries();
            load(first);
        }
        for (int it = first; it < end; ++it) {
            S::wait(0);
            barrier();
            if (it + 1 < end) load(it + 1);
            if (it >= mine) continue;
            scores(it);
            weights(it);
            values(it);
        }
    } else if (first < end) {
        // A wave asks for a tile so far ahead that all waves are done with the
        // one in its place: in their weights of tile `it`, the late waves know
        // the others to be past the values of it - 1, those know no more than
        // that the late ones are at them.
        const int ahead = NW == 1 || late ? STAGES - 1 : STAGES - 2;
        // Waits for this wave's part of tile `it`, where the next STAGES - 3
        // were asked for too.
        auto arrived = [&](int it) { S::wait(max(0, min(NW == 1 ? STAGES - 2 : STAGES - 3, end - 1 - it))); };
        constexpr int kBefore = NW == 1 ? STAGES - 1 : STAGES - 2;
        askQueries();
        for (int it = first; it < min(first + kBefore, end); ++it) load(it);
        if (PING) S::wait(min(kBefore, end - first));
        takeQueries();
        S::wait(max(0, min(kBefore, end - first) - 1));
        if (PING) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        if (late && first + kBefore < end) load(first + kBefore);
        if (first < mine) scores(first);
        if (late) {
            arrived(first + 1);
            barrier();
        }
        auto keep = [&](int it) {
            if (it + ahead < end) load(it + ahead);
        };
        auto before = [&](int it) {
            if (!late) arrived(it + 1);
            barrier();
            __builtin_amdgcn_s_setprio(1);
        };
        auto after = [&](int it) {
            __builtin_amdgcn_s_setprio(0);
            if (PING) {
                if (late) arrived(it + 2);
                barrier();
            }
        };
        int it = first;
        for (; it + 1 < mine; ++it) {
            keep(it);
            weights(it);
            before(it);
            values(it);
            scores(it + 1);
            if constexpr (sizeof(T) == 2) readAhead<S::kKeys / 16 * DB, KB * KS, 4>();
            after(it);
        }
        if (it < mine) {
            keep(it);
            weights(it);
            before(it);
            values(it);
            if constexpr (sizeof(T) == 2) readAhead<S::kKeys / 16 * DB, 0, 4>();
            after(it++);
        }
        for (; it < end; ++it) {
            keep(it);
            before(it);
            after(it);
        }
        if (PING && !late) barrier();
    }
    // A weight of 0 takes an infinite or NaN value to NaN: where a row came out
    // non-finite, the block is summed again key by key, hidden keys left out. Also
    // where f32 holds the maximum in steps of 2 or more: it is off the score it
    // was rounded from by up to half a step, and all weights by as many powers of
    // two. Key by key they are relative to scores rounded alike.
    float zero = fabsf(m) < kFar || m == kLowest ? 0.0f * l : NAN;
#pragma unroll
    for (int i = 0; i < DB; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) zero = __builtin_fmaf(o[i][e], 0.0f, zero);
    }
    if (__syncthreads_or(zero != 0.0f)) {   // NaN, where one was not finite
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = f32x16{};
        m = kLowest;
        l = 0.0f;
        next = start(first);
        for (int it = first; it < end; ++it) {
            load(it);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const char* tile = place(it);
            const int j0 = firstKey(it), seen = (it < tilesP ? np : lim) - j0;
            const int n = it < mine ? min((it < tilesP ? np : nk) - j0, S::kKeys) : 0;
            for (int j = 0; j < n; ++j) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const P kk = *reinterpret_cast<const P*>(tile + j * RB + (((2 * i + hl) ^ swizzleK<RB>(j)) << 4));
                    // This path is rare: no registers for its sake, so that
                    // its conversions of q stay where they are.
                    f32x4 bits = __builtin_bit_cast(f32x4, q[i]);
                    asm volatile("" : "+v"(bits));
                    const P qq = __builtin_bit_cast(P, bits);
#pragma unroll
                    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) s += static_cast<float>(qq[e]) * static_cast<float>(kk[e]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                s += otherHalf(s);
                if (j >= seen) s = -INFINITY;
                const float x = s * c, top = fmaxf(m, x - S::kTop), keep = __builtin_amdgcn_exp2f(m - top);
                const float u = __builtin_amdgcn_exp2f(x - top);
                m = top;
                l = l * keep + (hl == 0 ? u : 0.0f);
                const float ut = static_cast<float>(static_cast<T>(u));
#pragma unroll
                for (int i = 0; i < DB; ++i) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int byte = (32 * i + 2 * e + 4 * hl) * static_cast<int>(sizeof(T));
                        const V4 vv = *reinterpret_cast<const V4*>(tile + S::kTile + j * RB + (((byte >> 4) ^ swizzleV<T, RB>(j)) << 4) + (byte & 15));
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                            const float old = o[i][e + f] * keep;
                            o[i][e + f] = j < seen ? old + ut * static_cast<float>(vv[f]) : old;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            __syncthreads();
        }
    }

    // Results by whole rows through LDS, each wave its own 32 rows, 16 bytes a
    // lane (8 bytes of each of 64 rows at a time take 64 cycles a store).
    l += otherHalf(l);
    if constexpr (KG == 2) {   // the groups' sums joined, a lane's with its like's
        float* const at = reinterpret_cast<float*>(ldsTiles) + wave % (NW / 2) * (DB * 16 + 2) * 64 + ln;
        if (wave >= NW / 2) {
#pragma unroll
            for (int i = 0; i < DB; ++i) {
#pragma unroll
                for (int e = 0; e < 16; ++e) at[(i * 16 + e) * 64] = o[i][e];
            }
            at[DB * 16 * 64] = m;
            at[(DB * 16 + 1) * 64] = l;
        }
        __syncthreads();
        if (wave < NW / 2) {
            const float m1 = at[DB * 16 * 64], top = fmaxf(m, m1), keep = __builtin_amdgcn_exp2f(m - top), keep1 = __builtin_amdgcn_exp2f(m1 - top);
            m = top;
            l = l * keep + at[(DB * 16 + 1) * 64] * keep1;
#pragma unroll
            for (int i = 0; i < DB; ++i) {
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] = o[i][e] * keep + at[(i * 16 + e) * 64] * keep1;
            }
        }
        __syncthreads();
        if (wave >= NW / 2) return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (hl == 0 && rw + l32 < rows) {
        const int t = tokenOf(rw + l32), h = rw + l32 - (t + token0) * group + g * group;
        const int64_t row = (s.q0 + token0 + t) * p.heads + h;
        if (a.parts > 0) a.ml[static_cast<int64_t>(a.part0 + split) * p.q_rows * p.heads + row] = make_float2(m, l);
        else if (p.lse != nullptr) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
    auto store = [&](auto zero, float scale, auto rowAt) {
        using O = decltype(zero);
        constexpr int OB = RB / static_cast<int>(sizeof(T)) * static_cast<int>(sizeof(O)), OP = OB / 16, PER = 64 / OP;   // bytes and pieces of a row
        constexpr int SWIZZLE = OP < 16 ? OP - 1 : 15;
        static_assert(S::kRows * OB <= S::kLds && NW / 2 * (DB * 16 + 2) * 256 <= (KG == 2 ? S::kLds : 1 << 30), "the rows fit LDS");
        char* const at = ldsTiles + wave * 32 * OB;
#pragma unroll
        for (int i = 0; i < DB; ++i) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                Vec4<O> v;
#pragma unroll
                for (int f = 0; f < 4; ++f) v[f] = static_cast<O>(o[i][e + f] * scale);
                const int byte = (i * 32 + 2 * e + 4 * hl) * static_cast<int>(sizeof(O));
                *reinterpret_cast<Vec4<O>*>(at + l32 * OB + (((byte >> 4) ^ (l32 & SWIZZLE)) << 4) + (byte & 15)) = v;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 32 / PER; ++i) {
            const int row = i * PER + ln / OP, piece = ln % OP;
            const f32x4 v = *reinterpret_cast<const f32x4*>(at + row * OB + ((piece ^ (row & SWIZZLE)) << 4));
            if (rw + row < rows && piece * 16 < p.dim * static_cast<int>(sizeof(O))) *reinterpret_cast<f32x4*>(rowAt(rw + row) + piece * 16) = v;
        }
    };
    if (a.parts > 0) {
        char* const acc = reinterpret_cast<char*>(a.acc + static_cast<int64_t>(a.part0 + split) * p.q_rows * p.heads * p.dim);
        store(0.0f, 1.0f, [&](int r) {
            const int t = tokenOf(r);
            return acc + ((s.q0 + token0 + t) * p.heads + (r - (t + token0) * group + g * group)) * static_cast<int64_t>(p.dim) * 4;
        });
    } else {
        char* const out = reinterpret_cast<char*>(static_cast<T*>(p.out) + (s.q0 + token0) * p.out_stride);
        store(static_cast<T>(0.0f), inv, [&](int r) { return out + static_cast<uint64_t>(placeOf(r, p.out_stride)) * sizeof(T); });
    }
}

}  // namespace mlk
