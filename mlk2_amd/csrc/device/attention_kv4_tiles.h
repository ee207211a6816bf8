// Attention over a cache in 4 bits on matrix cores: a wave 32 query rows, over
// tiles of 32 keys.
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
    int units;                       // row blocks times key ranges
};

/// The numbers of a word's eight codes, exact in either type.
template <typename T>
__device__ __forceinline__ Piece<T> numbers(int word);
template <>
__device__ __forceinline__ Piece<__bf16> numbers<__bf16>(int word) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 3);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
template <>
__device__ __forceinline__ Piece<_Float16> numbers<_Float16>(int word) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 3);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

/// NW waves with the same 32 rows, the tiles in turn; their sums are joined at
/// the end.
template <typename T, int DT, int NW>
struct Kv4Tiles {
    using Q = std::conditional_t<std::is_same_v<T, float>, __bf16, T>;      // the scores' operands
    static constexpr int kPartsQ = std::is_same_v<T, float> ? 3 : 1;        // of a query: 24 bits in 8 each
    static constexpr int kPartsW = std::is_same_v<T, float> ? 3 : std::is_same_v<T, _Float16> ? 2 : 1;   // of a weight
    static constexpr int KS = DT / 16, DB = DT / 32;                        // steps of q k^T; 32-column blocks of out
    static constexpr int kWords = DT / 16;                                  // of a lane: half a key's codes
    static constexpr int kPiece = DT == 64 || DT == 128 ? 16 : 8;           // bytes of a load of codes; a head is whole ones
    static constexpr int kPitch = DT == 64 ? 48 : DT <= 128 ? 80 : 144;     // bytes from value row to row in LDS: 16 rows' words in different banks
    static constexpr int kTile = 32 * kPitch + 256;                         // a wave's values and scales
    static constexpr int kRow = DT * 4;                                     // bytes of a row of results
    static constexpr int kJoin = 32 * kRow + 256;
    static constexpr int kLds = NW * (kTile > kJoin ? kTile : kJoin);
};

/// Waves of a SIMD that the registers have to hold.
template <typename T>
constexpr int kv4Waves(int dt) {
    return std::is_same_v<T, float> || dt > 128 ? 1 : 2;
}

/// One row block of one key/value head. With S^T = K Q^T in 32 x 32 blocks a lane
/// holds 16 keys' scores of one query (the other 16 in lane ^ 32), so the softmax
/// is register work but for one exchange of maxima. The products run on the codes
/// as numbers, which either 16-bit type holds exactly: a key's scale goes to its
/// scores, a value's to its weights. Half a key row's codes are a lane's operand
/// as they lie in memory, eight to a word. Values take one trip through LDS: a
/// transposing read of 4-bit elements hands a lane one column of the 16 keys whose
/// weights it holds, in their order.
///
/// What is rounded: a weight times its value's scale to bf16 (f16 rows: to two
/// bf16 parts, 16 bits, f32 rows three), half a step of itself; f32 queries are
/// three bf16 parts, exactly. Scores, weights, their sum and out's sums are f32.
/// The maximum that the weights are relative to follows the running one only when
/// that has grown by 2^8.
template <typename T, int DT, int NW>
__global__ __launch_bounds__(NW * 64, kv4Waves<T>(DT)) void attentionKv4Tiles(Kv4Args args) {
    using S = Kv4Tiles<T, DT, NW>;
    using Q = typename S::Q;
    constexpr int KS = S::KS, DB = S::DB, WORDS = S::kWords;
    extern __shared__ __align__(16) char ldsTiles[];
    const TileArgs& a = args.t;
    const mlkd_attention& p = a.p;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int ln = threadIdx.x & 63, l32 = ln & 31, hl = ln >> 5;
    // The heads of a unit go to one XCD one after the other: neighbouring heads'
    // codes share lines of 128 bytes.
    const int id = static_cast<int>(blockIdx.x), turn = id / 8, upper = turn / a.by_kv_heads, g = turn - upper * p.kv_heads;
    const int unit = upper * 8 + id % 8;
    if (unit >= args.units) return;
    const int rest = unit / a.by_splits, split = unit - rest * a.splits, group = p.heads / p.kv_heads;
    SeqSpan s{};
    int r0 = 0;
    if (!rowBlock<32>(p, group, rest, s, r0)) return;
    s = SeqSpan{uniform(s.q0), uniform(s.k0), static_cast<int32_t>(uniform(s.nq)), static_cast<int32_t>(uniform(s.nk))};
    r0 = __builtin_amdgcn_readfirstlane(r0);
    const int rows = s.nq * group;
    // Keys that a row sees: those below its limit.
    auto limit = [&](int r) {
        return p.causal != 0 ? min(max(min(r, rows - 1) / a.by_group + s.nk - s.nq + 1, 0), s.nk) : s.nk;
    };
    const int limLo = __builtin_amdgcn_readfirstlane(limit(r0)), limHi = __builtin_amdgcn_readfirstlane(limit(r0 + 31)), lim = limit(r0 + l32);
    const int tiles = (limHi + 31) / 32, each = tiles / a.by_splits, more = tiles - each * a.splits;
    const int first = __builtin_amdgcn_readfirstlane(each * split + min(split, more)) + wave;
    const int end = __builtin_amdgcn_readfirstlane(each * split + min(split, more) + each + (split < more ? 1 : 0));
    const int token0 = __builtin_amdgcn_readfirstlane(r0 / a.by_group);
    auto tokenOf = [&](int r) { return r / a.by_group - token0; };
    auto headOf = [&](int r, int t) { return r - (t + token0) * group + g * group; };

    // Queries: step i takes elements hl DT / 2 + 8 i .. + 7, as half a key row lies.
    Piece<Q> q[S::kPartsQ][KS];
    {
        const int r = min(r0 + l32, rows - 1), t = tokenOf(r);
        const T* row = static_cast<const T*>(p.q) + (s.q0 + token0 + t) * p.q_stride + static_cast<int64_t>(headOf(r, t)) * p.dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int d = hl * (DT / 2) + 8 * i;
            using V8 = T __attribute__((ext_vector_type(8)));
            V8 v = {};
            if (d < p.dim) v = *reinterpret_cast<const V8*>(row + d);
            if constexpr (S::kPartsQ == 1) {
                q[0][i] = v;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float left = v[e];
#pragma unroll
                    for (int n = 0; n < S::kPartsQ; ++n) {
                        q[n][i][e] = static_cast<Q>(left);
                        left -= static_cast<float>(q[n][i][e]);
                    }
                }
            }
        }
    }
    const float c = static_cast<float>(p.scale * 1.4426950408889634);

    struct Tile {
        int k[WORDS], v[WORDS];
        float scale;   // a key's: of k in the lower half wave, of v in the upper
    };
    const int halfAt = hl * (DT / 4), bytes = p.dim / 2;
    // Pieces of the half row behind the head's end repeat its last: their queries
    // are zeros, their columns not stored.
    auto codes = [&](int (&to)[WORDS], const char* row) {
        using Words = int __attribute__((ext_vector_type(S::kPiece / 4)));
#pragma unroll
        for (int i = 0; i < WORDS; i += S::kPiece / 4) {
            const Words v = *reinterpret_cast<const Words*>(row + min(halfAt + 4 * i, bytes - S::kPiece));
#pragma unroll
            for (int e = 0; e < S::kPiece / 4; ++e) to[i + e] = v[e];
        }
    };
    const char *const k0 = static_cast<const char*>(p.k) + s.k0 * p.k_stride + static_cast<int64_t>(g) * bytes,
               *const v0 = static_cast<const char*>(p.v) + s.k0 * p.v_stride + static_cast<int64_t>(g) * bytes;
    const float* const scales = (hl == 0 ? args.k_scale : args.v_scale) + s.k0 * p.kv_heads + g;
    auto load = [&](int it, Tile& to) {
        const int64_t j0 = static_cast<int64_t>(it) * 32;
        const int j = min(l32, limHi - 1 - it * 32);   // keys behind the last repeat it
        codes(to.k, k0 + j0 * p.k_stride + static_cast<uint32_t>(j) * static_cast<uint32_t>(p.k_stride));
        codes(to.v, v0 + j0 * p.v_stride + static_cast<uint32_t>(j) * static_cast<uint32_t>(p.v_stride));
        to.scale = scales[(j0 + j) * p.kv_heads];
    };

    char* const mine = ldsTiles + wave * S::kTile;
    float* const tileScales = reinterpret_cast<float*>(mine + 32 * S::kPitch);
    // The row whose bytes this lane hands the transposing read, and its columns.
    const char* const column = mine + (8 * ((ln & 15) >> 2) + 4 * hl + (ln & 3)) * S::kPitch + ((ln >> 4) & 1) * 8;
    f32x16 o[DB] = {};
    float m = kLowest, l = 0.0f;   // what the weights of this lane's query are relative to; of this lane's keys, their sum
    // Tile `it`; its registers take tile `then`'s codes once they are used.
    auto process = [&](int it, Tile& tile, int then) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 2) *reinterpret_cast<i32x2*>(mine + l32 * S::kPitch + halfAt + 4 * i) = i32x2{tile.v[i], tile.v[i + 1]};
        tileScales[ln] = hl == 0 ? tile.scale * c : tile.scale;
        f32x16 x = {};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const Piece<Q> k = numbers<Q>(tile.k[i]);
#pragma unroll
            for (int n = 0; n < S::kPartsQ; ++n) x = mfma(k, q[n][i], x);
        }
        load(min(then, end - 1), tile);   // always: a wait for one tile's loads counts the next one's
        f32x4 ks[4], vs[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ks[e] = *reinterpret_cast<const f32x4*>(tileScales + 8 * e + 4 * hl);
            vs[e] = *reinterpret_cast<const f32x4*>(tileScales + 32 + 8 * e + 4 * hl);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= ks[e / 4][e % 4];
        const int seen = lim - it * 32 - 4 * hl;   // keys of this lane's, counted as the scores are
        const bool edge = limLo < it * 32 + 32;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 8 * (e / 4) + e % 4 < seen ? x[e] : -INFINITY;
            asm volatile("" : "+v"(x));   // a branch
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
        top = fmaxf(top, otherHalf(top));
        while (__any(top > m + 8.0f)) {   // once at most
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
        for (int e = 0; e < 16; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e] - m);
            l += x[e];
            x[e] *= vs[e / 4][e % 4];
        }
        if (edge) {   // a hidden value's scale may be anything
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 8 * (e / 4) + e % 4 < seen ? x[e] : 0.0f;
            asm volatile("" : "+v"(x));
        }
        Piece<__bf16> w[S::kPartsW][2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float left = x[e];
#pragma unroll
            for (int n = 0; n < S::kPartsW; ++n) {
                w[n][e / 8][e % 8] = static_cast<__bf16>(left);
                left -= static_cast<float>(w[n][e / 8][e % 8]);
            }
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            using Lds = __attribute__((address_space(3))) i32x2;
            const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32((Lds*)(column + i * 16));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const Piece<__bf16> vv = numbers<__bf16>(v[half]);
#pragma unroll
                for (int n = 0; n < S::kPartsW; ++n) o[i] = mfma(vv, w[n][half], o[i]);
            }
        }
    };
    if constexpr (DT <= 128) {   // two tiles in registers
        Tile one, two;
        if (first < end) load(first, one);
        if (first < end) load(min(first + NW, end - 1), two);
        for (int it = first; it < end; it += 2 * NW) {
            process(it, one, it + 2 * NW);
            if (it + NW >= end) break;
            process(it + NW, two, it + 3 * NW);
        }
    } else {
        Tile one;
        if (first < end) load(first, one);
        for (int it = first; it < end; it += NW) process(it, one, it + NW);
    }

    // The waves' sums by rows through LDS, 16 bytes a lane, joined on the way out.
    l += otherHalf(l);
    if constexpr (NW > 1) __syncthreads();   // all are done with their tiles
    char* const sums = ldsTiles;
    float2* const tops = reinterpret_cast<float2*>(ldsTiles + NW * 32 * S::kRow);
    if (r0 + l32 < rows) {
        char* const at = sums + (wave * 32 + l32) * S::kRow;
#pragma unroll
        for (int i = 0; i < DB; ++i) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int piece = i * 8 + 2 * (e / 4) + hl;
                *reinterpret_cast<f32x4*>(at + ((piece ^ (l32 & 7)) << 4)) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
            }
        }
        if (hl == 0) tops[wave * 32 + l32] = make_float2(m, l);
    }
    if constexpr (NW > 1) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    constexpr int LPR = DT <= 64 ? 16 : DT <= 128 ? 32 : 64, SIDE = 64 / LPR;   // lanes of a row, rows side by side
    const int piece = ln % LPR;
    for (int row = wave * SIDE + ln / LPR; row < min(32, rows - r0); row += NW * SIDE) {
        float2 ml[NW];
        float top = kLowest, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            ml[w] = tops[w * 32 + row];
            top = fmaxf(top, ml[w].x);
        }
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float keep = NW == 1 ? 1.0f : __builtin_amdgcn_exp2f(ml[w].x - top);
            sum += ml[w].y * keep;
            if (piece * 4 < DT) v += *reinterpret_cast<const f32x4*>(sums + (w * 32 + row) * S::kRow + ((piece ^ (row & 7)) << 4)) * keep;
        }
        const int t = tokenOf(r0 + row), h = headOf(r0 + row, t);
        const int64_t at = (s.q0 + token0 + t) * p.heads + h;
        if (piece == 0) {
            if (a.parts > 0) a.ml[static_cast<int64_t>(split) * p.q_rows * p.heads + at] = make_float2(top, sum);
            else if (p.lse != nullptr) p.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
        if (piece * 4 >= p.dim) continue;
        if (a.parts > 0) {
            *reinterpret_cast<f32x4*>(a.acc + (static_cast<int64_t>(split) * p.q_rows * p.heads + at) * p.dim + piece * 4) = v;
        } else {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            Vec4<T> out;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(v[e] * inv);
            *reinterpret_cast<Vec4<T>*>(static_cast<T*>(p.out) + (s.q0 + token0 + t) * p.out_stride + static_cast<int64_t>(h) * p.dim + piece * 4) = out;
        }
    }
}

}  // namespace mlk
