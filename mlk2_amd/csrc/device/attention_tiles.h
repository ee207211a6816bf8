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

/// What a launch of tiles works on: which keys, which rows, and where the
/// results go.
struct TileArgs {
    mlkd_attention p;
    int keys;         // 1: the prefix, 2: the sequences' own, 3: both
    int all_rows;     // 1: rows of all sequences together (prefix keys only)
    int splits;       // key ranges of each row block
    int part0;        // partial results: the first range's index ...
    int parts;        // ... of so many (0: results go straight to out)
    float* acc;       // [parts][rows * heads][dim]
    float2* ml;       // [parts][rows * heads]: maximum (times log2 e), sum
};

/// The row block `tile` counted from the end of the batch: its sequence and
/// first row. Rows are (token, head of the group); each sequence has
/// ceil(nq * group / rows) blocks. All lanes return the same; false past the
/// first block.
__device__ __forceinline__ bool rowBlock(const mlkd_attention& p, int group, int rows, int tile, int& b, int& r0) {
    const int ln = threadIdx.x & 63;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        const int s = p.sequences - 1 - s0 - ln;
        const int mine = s >= 0 ? (spanOf(p, s).nq * group + rows - 1) / rows : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d, 64);
            sum += ln >= d ? v : 0;
        }
        const uint64_t past = __ballot(sum > tile);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            b = __builtin_amdgcn_readfirstlane(p.sequences - 1 - s0 - at);
            r0 = __builtin_amdgcn_readfirstlane((__builtin_amdgcn_readlane(sum, at) - 1 - tile) * rows);
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

template <typename T, int DT, int NW, int KEYS, int STAGES>
struct Tiles {
    static constexpr int KS = DT * sizeof(T) / 32, DB = DT / 32;      // steps of q k^T, two pieces each; 32-column blocks of out
    static constexpr int RB = (DT <= 64 ? 64 : DT <= 128 ? 128 : 256) * sizeof(T);
    static constexpr int kTile = KEYS * RB;                          // bytes of a tile of keys
    static constexpr int kStage = 2 * kTile;
    static constexpr int kLds = STAGES * kStage;
    static constexpr int kRows = 32 * NW;
    static constexpr int IPW = kTile / 1024 / NW;                    // 1024-byte loads of a wave, for keys and again for values
    static constexpr int KB = KEYS / 32;
    static_assert(IPW >= 1 && IPW * NW * 1024 == kTile, "a tile is whole loads of the waves");
    static_assert(STAGES == 2 || (STAGES - 2) * 2 * IPW <= 63, "the loads waited on by number fit the counter");

    static __device__ __forceinline__ void dma(const void* base, uint32_t off, uint32_t m0) {
        asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
    }

    static __device__ __forceinline__ int swizzle(int half, int row) {
        return half == 0 ? swizzleK<RB>(row) : swizzleV<T, RB>(row);
    }

    /// This wave's loads of a tile, straight to LDS: rows past the last valid
    /// one repeat it; pieces past the head dim stay zero.
    static __device__ __forceinline__ void load(const void* k, const void* v, uint32_t ks, uint32_t vs, int last, int pieces, uint32_t lds, int wave) {
        constexpr int P = RB / 16, R = 64 / P;   // pieces of a row, rows of a load
        int ln = threadIdx.x & 63;
        asm volatile("" : "+v"(ln));   // the offsets are taken anew for each tile: kept, they are up to 64 registers
        if (last >= KEYS - 1 && pieces == P) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t stride = half == 0 ? ks : vs;
                const char* base = static_cast<const char*>(half == 0 ? k : v) + static_cast<uint64_t>(wave * IPW * R) * stride;
                const uint32_t row = ln / P * stride, piece = ((ln % P) ^ swizzle(half, wave * IPW * R + ln / P)) << 4;
#pragma unroll
                for (int i = 0; i < IPW; ++i) {
                    // Rows i R + r with r < R: their swizzle is i R's and r's.
                    const int w0 = wave * IPW * R, turned = swizzle(half, w0 + i * R) ^ swizzle(half, w0);
                    dma(base + static_cast<uint64_t>(i * R) * stride, (piece ^ (turned << 4)) + row, lds + half * kTile + (wave * IPW + i) * 1024);
                }
            }
            return;
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
#pragma unroll 1
            for (int i = 0; i < IPW; ++i) {
                const int n = wave * IPW + i, row = n * R + ln / P, piece = (ln % P) ^ swizzle(half, row);
                const uint32_t off = static_cast<uint32_t>(min(row, last)) * (half == 0 ? ks : vs) + piece * 16;
                if (piece < pieces) dma(half == 0 ? k : v, off, lds + half * kTile + n * 1024);
            }
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
/// up to 2^8 lose nothing in f32, and out is rescaled in few tiles.
template <typename T, int DT, int NW, int KEYS, int STAGES>
__global__ __launch_bounds__(NW * 64, DT > 128 ? 1 : 2) void attentionTiles(TileArgs a) {
    using S = Tiles<T, DT, NW, KEYS, STAGES>;
    using P = Piece<T>;
    using V4 = Vec4<T>;
    using Short4 = short __attribute__((ext_vector_type(4)));
    constexpr int KS = S::KS, DB = S::DB, RB = S::RB, KB = S::KB;
    constexpr bool PING = NW == 8;
    extern __shared__ __align__(16) char ldsTiles[];
    const mlkd_attention& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int ln = threadIdx.x & 63, l32 = ln & 31, hl = ln >> 5;
    const int group = p.heads / p.kv_heads, g = static_cast<int>(blockIdx.x) % p.kv_heads;
    int rest = static_cast<int>(blockIdx.x) / p.kv_heads;
    const int split = rest % a.splits;
    rest /= a.splits;
    SeqSpan s;
    int r0 = 0;
    if (a.all_rows != 0) {
        s = SeqSpan{0, 0, static_cast<int32_t>(p.q_rows), 0};
        r0 = rest * S::kRows;
        if (r0 >= s.nq * group) return;
    } else {
        int b = 0;
        if (!rowBlock(p, group, S::kRows, rest, b, r0)) return;
        s = spanOf(p, b);
    }
    const int rows = s.nq * group;
    // Keys that a row sees: the prefix, and own keys below lim = token + slope.
    const int np = (a.keys & 1) != 0 ? prefixOf(p) : 0, nk = (a.keys & 2) != 0 ? s.nk : 0;
    auto limit = [&](int r) {
        return p.causal != 0 ? min(max(min(r, rows - 1) / group + s.nk - s.nq + 1, 0), nk) : nk;
    };
    const int tilesP = (np + KEYS - 1) / KEYS, tiles = tilesP + (limit(r0 + S::kRows - 1) + KEYS - 1) / KEYS;
    const int first = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits));
    const int end = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits));
    const int rw = r0 + wave * 32;                       // this wave's first row
    const int limLo = limit(rw), limHi = limit(rw + 31);
    const int r = min(rw + l32, rows - 1), lim = limit(r), head = g * group + r % group;
    const bool valid = rw + l32 < rows;
    const int64_t token = s.q0 + r / group;

    // Queries, a piece a step; a negative scale turns their signs.
    const float c = static_cast<float>(fabs(p.scale) * 1.4426950408889634);
    P q[KS];
    {
        const T* qr = static_cast<const T*>(p.q) + token * p.q_stride + static_cast<int64_t>(head) * p.dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int d = (2 * i + hl) * (16 / static_cast<int>(sizeof(T)));
            P x = {};
            if (d < p.dim) x = *reinterpret_cast<const P*>(qr + d);
            if (p.scale < 0.0) x = -x;
            q[i] = x;
        }
    }

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ldsTiles));
    const int pieces = p.dim * static_cast<int>(sizeof(T)) / 16;
    if (p.dim < DT) {   // what the loads leave out
        for (int i = threadIdx.x * 16; i < S::kLds; i += NW * 64 * 16) *reinterpret_cast<f32x4*>(ldsTiles + i) = f32x4{};
        __syncthreads();
    }
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
        S::load(next.k, next.v, next.ks, next.vs, next.left - 1, pieces, lds0 + next.at, wave);
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
    float m = kLowest, l = 0.0f;   // of this lane's query; l of this lane's keys
    auto place = [&](int it) { return ldsTiles + (it - first) % STAGES * S::kStage; };
    auto firstKey = [&](int it) { return (it < tilesP ? it : it - tilesP) * KEYS; };
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
    P w[sizeof(T) == 4 ? 1 : KEYS / 16];
    auto weights = [&](int it) {
        const int j0 = firstKey(it);
        if ((it < tilesP ? np : limLo) < j0 + KEYS) {
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
        top = fmaxf(top, otherHalf(top)) * c;
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
            for (int kg = 0; kg < KEYS / 16; ++kg) {
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
            for (int kg = 0; kg < KEYS / 16; ++kg) {
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
        if (first < end) load(first);
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
        for (int it = first; it < min(first + ahead, end); ++it) load(it);
        S::wait(max(0, min(ahead, end - first) - 1));
        barrier();
        if (first < mine) scores(first);
        if (late) {
            arrived(first + 1);
            barrier();
        }
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
            if (it + ahead < end) load(it + ahead);
            weights(it);
            before(it);
            values(it);
            scores(it + 1);
            if constexpr (sizeof(T) == 2) readAhead<KEYS / 16 * DB, KB * KS, 4>();
            after(it);
        }
        if (it < mine) {
            if (it + ahead < end) load(it + ahead);
            weights(it);
            before(it);
            values(it);
            if constexpr (sizeof(T) == 2) readAhead<KEYS / 16 * DB, 0, 4>();
            after(it++);
        }
        for (; it < end; ++it) {
            if (it + ahead < end) load(it + ahead);
            before(it);
            after(it);
        }
        if (PING && !late) barrier();
    }
    // A weight of 0 takes an infinite or NaN value to NaN: where a row came out
    // non-finite, the block is summed again key by key, hidden keys left out.
    bool bad = !(fabsf(l) < INFINITY);
#pragma unroll
    for (int i = 0; i < DB; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) bad |= !(fabsf(o[i][e]) < INFINITY);
    }
    if (__syncthreads_or(bad)) {
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
            const int n = it < mine ? min((it < tilesP ? np : nk) - j0, KEYS) : 0;
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
                const float top = fmaxf(m, s * c), keep = __builtin_amdgcn_exp2f(m - top);
                const float u = __builtin_amdgcn_exp2f(s * c - top);
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

    l += otherHalf(l);
    if (!valid) return;
    const int64_t row = token * p.heads + head;
    if (a.parts > 0) {
        const int64_t at = static_cast<int64_t>(a.part0 + split) * p.q_rows * p.heads + row;
        if (hl == 0) a.ml[at] = make_float2(m, l);
        float* out = a.acc + at * p.dim;
#pragma unroll
        for (int i = 0; i < DB; ++i) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = i * 32 + 2 * e + 4 * hl;
                if (d < p.dim) *reinterpret_cast<f32x4*>(out + d) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
            }
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(p.out) + token * p.out_stride + static_cast<int64_t>(head) * p.dim;
#pragma unroll
    for (int i = 0; i < DB; ++i) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = i * 32 + 2 * e + 4 * hl;
            V4 v;
#pragma unroll
            for (int f = 0; f < 4; ++f) v[f] = static_cast<T>(o[i][e + f] * inv);
            if (d < p.dim) *reinterpret_cast<V4*>(out + d) = v;
        }
    }
    if (p.lse != nullptr && hl == 0) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace mlk
