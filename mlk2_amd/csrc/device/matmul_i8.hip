// Products of rows in 8-bit integers, out = (a b^T) a_scale b_scale + bias: exact
// sums in 32 bits, turned to f32 and scaled as they are stored.
//
// v_mfma_i32_16x16x64_i8 takes 16 bytes a lane of either operand, 64 bytes of k
// of 16 rows, and both operands have their k along their rows, so that a wave's
// 16-byte pieces are its fragments as they stand. Operand b is the instruction's
// first: a lane then holds four neighbouring columns of one row of out.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "runtime_abi.h"
#include "xcd.h"

namespace {

using i32x4 = int __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;     // bytes of k that an instruction takes

__device__ __align__(16) const uint32_t kZero16[4] = {0u, 0u, 0u, 0u};

__device__ __forceinline__ i32x4 mfma(i32x4 b, i32x4 a, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, c, 0, 0, 0); }

/// 16 bytes at `from`, of any alignment, of which `left` are there; the others
/// are zeros.
__device__ __forceinline__ i32x4 piece(const int8_t* from, int64_t left) {
    i32x4 v = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (left >= 4 * i + 4) {
            int word;
            __builtin_memcpy(&word, from + 4 * i, 4);
            v[i] = word;
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                if (left > 4 * i + e) v[i] |= static_cast<int>(static_cast<uint8_t>(from[4 * i + e])) << e * 8;
            }
        }
    }
    return v;
}

/// 16 bytes of any alignment by whole words: reads off 4 bytes take three to five
/// times as long (64 x 8000 x 4095: 55 us, 4092: 22). The five words around them, or
/// the bytes as they are where a word reaches out of the operand, [lo, hi).
struct Window {
    i32x4 words;
    int last;
};
__device__ __forceinline__ bool whole(const int8_t* from, const int8_t* lo, const int8_t* hi) {
    const int8_t* base = from - (reinterpret_cast<uintptr_t>(from) & 3);
    return base >= lo && base + 20 <= hi;
}
__device__ __forceinline__ Window ask(const int8_t* from, const int8_t* lo, const int8_t* hi) {
    const bool in = whole(from, lo, hi);
    const int8_t* base = in ? from - (reinterpret_cast<uintptr_t>(from) & 3) : from;
    Window w;
    __builtin_memcpy(&w.words, base, 16);
    __builtin_memcpy(&w.last, base + (in ? 16 : 12), 4);
    return w;
}
__device__ __forceinline__ i32x4 take(const Window& w, const int8_t* from, const int8_t* lo, const int8_t* hi) {
    const int shift = whole(from, lo, hi) ? static_cast<int>(reinterpret_cast<uintptr_t>(from) & 3) : 0;
    i32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? w.words[i + 1] : w.last, w.words[i], shift);
    return v;
}

/// A row's scale as 2^-91 to 2^90 times a power of two, which comes last: a sum times
/// the one and the other operand's scale is in f32's range then where the result is.
struct RowScale {
    float s, rest;
};
__device__ __forceinline__ RowScale rowScale(float s) {
    const int e = __builtin_amdgcn_frexp_expf(s), by = e - max(-90, min(e, 90));
    return {__builtin_amdgcn_ldexpf(s, -by), __builtin_amdgcn_ldexpf(1.0f, by)};
}

template <typename T>
__device__ __forceinline__ T scaled(int sum, const RowScale& sa, float sb, float bias, bool has) {
    float v = static_cast<float>(sum) * sa.s * sb * sa.rest;
    if (has) v += bias;
    return static_cast<T>(v);
}

/// Columns n .. n + 3 of row m from their sums, n a multiple of 4. `wide`: rows
/// of whole 16-byte pieces at 16 bytes.
template <typename T>
__device__ __forceinline__ void store4(const mlkd_matmul_i8& p, int64_t m, int64_t n, i32x4 sum, const RowScale& sa, bool wide) {
    using V = T __attribute__((ext_vector_type(4)));
    T* out = static_cast<T*>(p.out) + m * p.ldo + n;
    const bool has = p.bias != nullptr;
    if (wide && n + 4 <= p.n) {
        V v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled<T>(sum[e], sa, p.b_scale[n + e], has ? p.bias[n + e] : 0.0f, has);
        *reinterpret_cast<V*>(out) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (n + e < p.n) out[e] = scaled<T>(sum[e], sa, p.b_scale[n + e], has ? p.bias[n + e] : 0.0f, has);
    }
}

// ------------------------------------------------------------- few rows ----
/// Blocks of 16 MB rows of a: eight waves take the 256-byte pieces of k in turn, 16
/// NB rows of b straight from memory, and their sums are added in LDS. A launch
/// reads b once and nothing waits but on those reads.
/// ALIGNED: rows at 4 bytes.
template <typename T, int MB, int NB, bool ALIGNED>
__global__ __launch_bounds__(512) void matmulI8Few(mlkd_matmul_i8 p, int wide) {
    constexpr int U = 4;   // steps of a piece
    const int8_t *endA = p.a + (p.m - 1) * p.lda + p.k, *endB = p.b + (p.n - 1) * p.ldb + p.k;
    __shared__ i32x4 sums[8][MB * NB][64];
    const int ln = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int l16 = ln & 15, g = ln >> 4;
    const int64_t blocks = (p.n + 16 * NB - 1) / (16 * NB);
    for (int64_t block = xcdShare(blockIdx.x, gridDim.x); block < blocks; block += gridDim.x) {
        const int64_t n0 = block * (16 * NB);
        const int64_t rows = blockIdx.y * int64_t{16 * MB};
        const int8_t *a[MB], *b[NB];
#pragma unroll
        for (int i = 0; i < MB; ++i) a[i] = p.a + min(rows + i * 16 + l16, p.m - 1) * p.lda + g * 16;
#pragma unroll
        for (int i = 0; i < NB; ++i) b[i] = p.b + min(n0 + i * 16 + l16, p.n - 1) * p.ldb + g * 16;
        i32x4 acc[MB][NB] = {};
        for (int64_t k = wave * (U * kStep); k < p.k; k += 8 * U * kStep) {
            i32x4 av[U][MB], bv[U][NB];
            if (k + U * kStep <= p.k && ALIGNED) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) __builtin_memcpy(&bv[u][i], b[i] + k + u * kStep, 16);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int i = 0; i < MB; ++i) __builtin_memcpy(&av[u][i], a[i] + k + u * kStep, 16);
                }
            } else if (k + U * kStep <= p.k) {
                Window aw[U][MB], bw[U][NB];
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) bw[u][i] = ask(b[i] + k + u * kStep, p.b, endB);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int i = 0; i < MB; ++i) aw[u][i] = ask(a[i] + k + u * kStep, p.a, endA);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) bv[u][i] = take(bw[u][i], b[i] + k + u * kStep, p.b, endB);
#pragma unroll
                    for (int i = 0; i < MB; ++i) av[u][i] = take(aw[u][i], a[i] + k + u * kStep, p.a, endA);
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t left = p.k - k - u * kStep - g * 16;
#pragma unroll
                    for (int i = 0; i < NB; ++i) bv[u][i] = piece(b[i] + k + u * kStep, left);
#pragma unroll
                    for (int i = 0; i < MB; ++i) av[u][i] = piece(a[i] + k + u * kStep, left);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < MB; ++i) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] = mfma(bv[u][j], av[u][i], acc[i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
#pragma unroll
            for (int j = 0; j < NB; ++j) sums[wave][i * NB + j][ln] = acc[i][j];
        }
        __syncthreads();
        for (int t = wave; t < MB * NB; t += 8) {
            i32x4 sum = sums[0][t][ln];
#pragma unroll
            for (int w = 1; w < 8; ++w) sum += sums[w][t][ln];
            const int64_t m = rows + t / NB * 16 + l16, n = n0 + t % NB * 16 + 4 * g;
            if (m < p.m && n < p.n) store4<T>(p, m, n, sum, rowScale(p.a_scale[m]), wide != 0);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- tiles ----
struct TileArgs {
    mlkd_matmul_i8 p;
    int tilesM, tilesN, splits, wide;
    int* work;     // [splits][m][ldw] sums of the ranges of k, or NULL
    int64_t ldw;   // n in whole fours
};

/// A tile of WM x WN waves of MT x NT products of 16 x 16 each, over steps of 64
/// bytes of k through a ring of kStages in LDS.
///
/// Rows of a and b, whole 16-byte pieces at 16 bytes, go straight to LDS, a ring of
/// steps ahead. The smaller tiles, with less to do a step, have longer rings and ask
/// for two steps at once, which fetches whole lines: 64 x 8000 of k = 4096 by 64 x 64,
/// b from memory, takes 24.3 us with a ring of four, 17.4 with one of eight, 15.7 by
/// two steps. Rows past the last repeat it, pieces past k are zeros.
///
/// LDS holds 64-byte rows, piece c of row r at c ^ (r / 4 % 4): a fragment's
/// read takes one piece of 16 rows at a time, which then lie in all banks. In
/// each step the products go in two halves: while the first runs, the second's
/// rows of a are read; while the second runs, the next step's fragments are read
/// and a later step's loads are asked for, in a fixed order, a memory
/// instruction behind every other product or so.
template <typename T, int WM, int WN, int MT, int NT, int kStages>
__global__ __launch_bounds__(WM * WN * 64, 2) void matmulI8Tiles(TileArgs args) {
    constexpr int NW = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16;
    constexpr int kStage = (BM + BN) * kStep, LOADS = (BM + BN) / 16 / NW, HM = MT / 2;
    constexpr bool PAIRS = kStages > 4;
    constexpr int kAhead = kStages - (PAIRS ? 2 : 1);   // the first steps asked for
    static_assert(LOADS * NW * 16 == BM + BN && HM * 2 == MT, "whole loads and halves");
    extern __shared__ __align__(16) char lds[];
    const mlkd_matmul_i8& p = args.p;
    const int ln = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int l16 = ln & 15, g = ln >> 4, wm = wave / WN, wn = wave % WN;
    // Tiles by XCD, those of one in bands of four tile rows.
    const int id = xcdShare(blockIdx.x, gridDim.x), split = id % args.splits, tile = id / args.splits;
    const int band = tile / (4 * args.tilesN), rest = tile - band * 4 * args.tilesN, high = min(4, args.tilesM - band * 4);
    const int64_t row0 = static_cast<int64_t>(band * 4 + rest % high) * BM, col0 = static_cast<int64_t>(rest / high) * BN;
    const int all = static_cast<int>((p.k + kStep - 1) / kStep);
    const int first = static_cast<int>(static_cast<int64_t>(all) * split / args.splits);
    const int steps = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / args.splits) - first;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));

    // This wave's loads of a step: 16 rows of 64 bytes each, of a's rows then b's.
    // A lane's piece lies `off` past its tile's first row.
    const int8_t* const tileA = p.a + row0 * p.lda + static_cast<int64_t>(first) * kStep;
    const int8_t* const tileB = p.b + col0 * p.ldb + static_cast<int64_t>(first) * kStep;
    uint32_t off[LOADS];
    const int at = ((ln & 3) ^ (ln >> 4)) * 16;   // the piece's first byte of k in a step
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (wave * LOADS + j) * 16 + (ln >> 2);
        const int64_t r = row < BM ? min(row0 + row, p.m - 1) - row0 : min(col0 + row - BM, p.n - 1) - col0;
        off[j] = static_cast<uint32_t>(r * (row < BM ? p.lda : p.ldb)) + at;
    }
    const int tail = static_cast<int>(p.k % kStep);   // bytes of the last step, or 0: all
    const bool partial = tail != 0 && first + steps == all;
    constexpr auto yes = [] { return true; };
    constexpr auto no = [] { return false; };
    // Load j of step t (past the last: the last again) into slot `slot`. `ends`:
    // that step may be the last.
    auto issue = [&](int t, int slot, int j, auto ends) __attribute__((always_inline)) {
        const int8_t* src = ((wave * LOADS + j) * 16 < BM ? tileA : tileB) + static_cast<int64_t>(ends() ? min(t, steps - 1) : t) * kStep;
        const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds0 + slot * kStage + (wave * LOADS + j) * 1024);
        if (ends() && partial && t >= steps - 1) {
            const int8_t* from = at < tail ? src + off[j] : reinterpret_cast<const int8_t*>(kZero16);
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(m0) : "memory");
        } else {
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[j]), "s"(src), "s"(m0) : "memory");
        }
    };
    i32x4 acc[MT][NT] = {};
    const uint32_t turn = (g ^ (l16 >> 2)) << 4;
    const uint32_t atA = lds0 + (wm * MT * 16 + l16) * kStep + turn, atB = lds0 + (BM + wn * NT * 16 + l16) * kStep + turn;
    constexpr int HS = kStages / 2;
    const uint32_t atA2 = atA + HS * kStage, atB2 = atB + HS * kStage;   // an instruction's offset holds 16 bits
    auto readA = [&](int slot, int i) {
        return *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>((slot < HS ? atA : atA2) + static_cast<uint32_t>(slot % HS * kStage + i * 16 * kStep));
    };
    auto readB = [&](int slot, int i) {
        return *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>((slot < HS ? atB : atB2) + static_cast<uint32_t>(slot % HS * kStage + i * 16 * kStep));
    };
    // Waits for all of this wave's loads but those of `later` steps.
    auto landed = [&](auto later) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(later() * LOADS) : "memory");
        asm volatile("s_barrier" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) issue(t, t, j, yes);
    }
    landed([] { return kAhead - 1; });
    i32x4 aLo[HM], aHi[HM], bX[NT], bY[NT];
#pragma unroll
    for (int i = 0; i < HM; ++i) aLo[i] = readA(0, i);
#pragma unroll
    for (int i = 0; i < NT; ++i) bX[i] = readB(0, i);
    // Step s in slot q. In pairs: an even step asks for two, an odd one for none.
    auto step = [&](int s, const int q, i32x4 (&bCur)[NT], i32x4 (&bNext)[NT], auto ends) __attribute__((always_inline)) {
        constexpr int N = HM * NT;
        const int next = (q + 1) % kStages;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int i = x / NT, j = (i & 1) != 0 ? NT - 1 - x % NT : x % NT;
            acc[i][j] = mfma(bCur[j], aLo[i], acc[i][j]);
#pragma unroll
            for (int r = 0; r < HM; ++r) {
                if (r * N / (2 * HM) == x) aHi[r] = readA(q, HM + r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // Step s + 1 is in LDS; every wave is past step s - 1, whose slot is free.
        landed([] { return kAhead - 2; });   // of two asked for at once, both
        __builtin_amdgcn_sched_barrier(0);
        constexpr int READS = NT + HM;   // B 0, A 0, the other Bs, the other As
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int i = x / NT, j = (i & 1) != 0 ? NT - 1 - x % NT : x % NT;
            acc[HM + i][j] = mfma(bCur[j], aHi[i], acc[HM + i][j]);
#pragma unroll
            for (int r = 0; r < READS; ++r) {
                if (r * N / READS != x) continue;
                if (r == 0) bNext[0] = readB(next, 0);
                else if (r == 1) aLo[0] = readA(next, 0);
                else if (r <= NT) bNext[r - 1] = readB(next, r - 1);
                else aLo[r - NT] = readA(next, r - NT);
            }
#pragma unroll
            for (int l = 0; l < (PAIRS ? 2 * LOADS : LOADS); ++l) {
                constexpr int ALL = PAIRS ? 2 * LOADS : LOADS;
                const int ahead = PAIRS ? kAhead + l % 2 : kAhead;
                if ((2 * l + 1) * N / (2 * ALL) != x || (PAIRS && (q & 1) != 0)) continue;
                issue(s + ahead, (q + ahead) % kStages, PAIRS ? l / 2 : l, ends);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int s = 0;
    // The slots' steps, from s on.
    auto round = [&](auto ends) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < kStages; q += 2) {
            if (ends() && s + q >= steps) break;
            step(s + q, q, bX, bY, ends);
            if (ends() && s + q + 1 >= steps) break;
            step(s + q + 1, q + 1, bY, bX, ends);
        }
        s += kStages;
    };
    while (s + 2 * (kStages - 1) < steps - 1) round(no);
    while (s < steps) round(yes);
    // No load may still be writing LDS, and no wave be reading it, when its rows
    // of results take its place.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // By whole rows through LDS, each wave its own, 16 bytes a lane (four columns
    // of 16 rows at a time, as the sums are held, took 15 us for 4096^2 f16 where
    // this takes 9).
    const int64_t m0 = row0 + wm * MT * 16, n0 = col0 + wn * NT * 16;
    auto store = [&](auto zero, bool wide, auto value, auto rowAt) __attribute__((always_inline)) {
        using O = decltype(zero);
        using V4 = O __attribute__((ext_vector_type(4)));
        constexpr int SIZE = sizeof(O), E = 16 / SIZE, PITCH = NT * 16 * SIZE, PIECES = PITCH / 16, PER = 64 / PIECES;
        constexpr int CHUNK = MT * 16 * PITCH * NW <= kStage * kStages ? MT : MT / 2;   // 16 rows each
        static_assert(CHUNK * 16 * PITCH * NW <= kStage * kStages && MT % CHUNK == 0, "the rows fit LDS");
        char* const mine = lds + wave * (CHUNK * 16 * PITCH);
#pragma unroll
        for (int i0 = 0; i0 < MT; i0 += CHUNK) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) {
                    const int byte = (j * 16 + 4 * g) * SIZE;
                    const V4 v = value(i0 + i, j, acc[i0 + i][j]);
                    *reinterpret_cast<V4*>(mine + (i * 16 + l16) * PITCH + (((byte >> 4) ^ (l16 & (PIECES - 1))) << 4) + (byte & 15)) = v;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int r = 0; r < CHUNK * 16 / PER; ++r) {
                const int row = r * PER + ln / PIECES, c = ln % PIECES;
                using V = O __attribute__((ext_vector_type(E)));
                const V v = *reinterpret_cast<const V*>(mine + row * PITCH + ((c ^ (row & 15 & (PIECES - 1))) << 4));
                const int64_t m = m0 + i0 * 16 + row, n = n0 + c * E;
                if (m >= p.m) continue;
                O* to = rowAt(m) + n;
                if (wide && n + E <= p.n) {
                    *reinterpret_cast<V*>(to) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (n + e < p.n) to[e] = v[e];
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    };
    if (args.splits > 1) {
        store(0, true, [&](int, int, i32x4 sum) { return sum; }, [&](int64_t m) { return args.work + (split * p.m + m) * args.ldw; });
        return;
    }
    RowScale sa[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sa[i] = rowScale(p.a_scale[min(m0 + i * 16 + l16, p.m - 1)]);
    store(static_cast<T>(0.0f), args.wide != 0, [&](int i, int j, i32x4 sum) {
        T __attribute__((ext_vector_type(4))) v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t n = min(n0 + j * 16 + 4 * g + e, p.n - 1);
            v[e] = scaled<T>(sum[e], sa[i], p.b_scale[n], p.bias != nullptr ? p.bias[n] : 0.0f, p.bias != nullptr);
        }
        return v;
    }, [&](int64_t m) { return static_cast<T*>(p.out) + m * p.ldo; });
}

/// Rows of k bytes copied to rows of `pitch` bytes at 16, zeros behind them: a's,
/// then b's. A thread a piece of 16 bytes.
__global__ __launch_bounds__(256) void matmulI8Pack(mlkd_matmul_i8 p, int8_t* to, int64_t pitch) {
    const int8_t *endA = p.a + (p.m - 1) * p.lda + p.k, *endB = p.b + (p.n - 1) * p.ldb + p.k;
    const int64_t pieces = pitch / 16, total = (p.m + p.n) * pieces;
    for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / pieces, c = (i - r * pieces) * 16;
        const bool inA = r < p.m;
        const int8_t *from = (inA ? p.a + r * p.lda : p.b + (r - p.m) * p.ldb) + c, *lo = inA ? p.a : p.b, *hi = inA ? endA : endB;
        *reinterpret_cast<i32x4*>(to + i * 16) = p.k - c >= 16 ? take(ask(from, lo, hi), from, lo, hi) : piece(from, p.k - c);
    }
}

/// The ranges' sums added, scaled and stored, four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void matmulI8Join(TileArgs args) {
    const mlkd_matmul_i8& p = args.p;
    const int64_t quads = args.ldw / 4, total = p.m * quads;
    for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        i32x4 sum = {};
        for (int s = 0; s < args.splits; ++s) sum += reinterpret_cast<const i32x4*>(args.work)[s * total + i];
        const int64_t m = i / quads;
        store4<T>(p, m, (i - m * quads) * 4, sum, rowScale(p.a_scale[m]), args.wide != 0);
    }
}

// --------------------------------------------------------------- launch ----
enum Form { kFew, kTile64, kTile128x64, kTile128, kTile256 };

/// A tile's rows and columns, what a round of 256 of them, one a unit, adds to the time
/// of k = 4096, in halves of a microsecond, and its threads.
struct TileSize {
    int rows, cols, round, threads;
};
constexpr TileSize kTiles[] = {{}, {64, 64, 16, 256}, {128, 64, 25, 256}, {128, 128, 40, 256}, {256, 256, 104, 512}};

struct Plan {
    Form form{kFew};
    bool aligned{false}, wide{false}, pack{false};
    int mb{1}, nb{1};      // kFew: 16 rows of a, of b, a workgroup
    int64_t tilesM{0}, tilesN{0};
    int splits{1}, stages{4};
};

int outBytes(const mlkd_matmul_i8* p) { return p->dtype == MLKD_F32 ? 4 : 2; }

/// Rows of whole pieces of so many bytes.
bool rowsAt(const mlkd_matmul_i8* p, int bytes) {
    return p->lda % bytes == 0 && p->ldb % bytes == 0 && reinterpret_cast<uintptr_t>(p->a) % bytes == 0 &&
           reinterpret_cast<uintptr_t>(p->b) % bytes == 0;
}

int64_t pitchOf(const mlkd_matmul_i8* p) { return (p->k + kStep - 1) / kStep * kStep; }

/// The workspace: the copied rows, then the ranges' sums.
int64_t packBytes(const mlkd_matmul_i8* p, const Plan& n) { return n.pack ? (p->m + p->n) * pitchOf(p) : 0; }
int64_t sumBytes(const mlkd_matmul_i8* p, const Plan& n) {
    return n.splits > 1 ? n.splits * p->m * ((p->n + 3) / 4 * 4) * static_cast<int64_t>(sizeof(int)) : 0;
}

/// `room`: with the workspace that it asks for.
Plan planOf(const mlkd_matmul_i8* p, bool room) {
    Plan n;
    const int size = outBytes(p);
    n.wide = p->ldo * size % 16 == 0 && reinterpret_cast<uintptr_t>(p->out) % 16 == 0;
    // A tile's rows lie 2^32 bytes apart at most.
    n.aligned = p->k % 16 == 0 && rowsAt(p, 16) && std::max(p->lda, p->ldb) < (int64_t{1} << 23);
    // (Here and below: us, b from memory rather than a cache, bf16 out.) Few rows go
    // without LDS while that is faster, in one round of workgroups of 32 columns.
    // Without and with, 32 x 8000 of k = 4096: 11.1 and 13.5, 32 x 2048 of 8192 13.6
    // and 11.7, 32 x 16384 of 4096 20.0 and 17.6; 64 x 8000 of 4096 14.9 and 13.6, of
    // 2048 9.4 and 9.6, 64 x 2048 of 2048 7.6 and 9.2, 64 x 12800 of 1024 11.4 and 7.2.
    const bool few = p->m <= 16 || (p->m <= 64 && (!n.aligned || (p->n <= 8192 && (p->m <= 32 ? p->k < 8192 : p->k <= 2048))));
    // A launch holds fewer than 2^32 threads.
    auto fits = [&](Form f) {
        return ((p->m + kTiles[f].rows - 1) / kTiles[f].rows) * ((p->n + kTiles[f].cols - 1) / kTiles[f].cols) < (int64_t{1} << 32) / kTiles[f].threads;
    };
    const bool tiles = !few && fits(kTile256);
    // The tiles take rows at 16 bytes: others are copied to such first.
    n.pack = !n.aligned && tiles && room;
    if (!tiles || !(n.aligned || n.pack)) {
        n.mb = p->m <= 16 ? 1 : p->m <= 32 ? 2 : 4;
        n.aligned = rowsAt(p, 4);
        // 32 of b's rows a workgroup where that still makes 200: 16 x 8000 of k = 4096
        // in 9.3, by 16 in 10.5; 16 x 4096 in 8.4, by 16 in 6.7.
        n.nb = p->n >= 32 * 200 ? 2 : 1;
        return n;
    }
    // The size whose rounds over 256 units take least. Of k = 4096, 256 x 4096 by
    // 64 x 64 takes 14.7 and by 128 x 64 20.3; 512 x 4096 22.8, 20.5 and by 128 x 128
    // 27.6; 512 x 8192 42.2, 34.9 and 28.9; 2048 x 4096 by 128 x 64 60.6, by 128 x 128
    // 50.5 and by 256 x 256 54.7; 2560 x 4096 63.5 and 56.6, 4096^2 98.8 and 65.2.
    int64_t best = INT64_MAX;
    for (Form f : {kTile64, kTile128x64, kTile128, kTile256}) {
        const int64_t rows = (p->m + kTiles[f].rows - 1) / kTiles[f].rows, cols = (p->n + kTiles[f].cols - 1) / kTiles[f].cols;
        const int64_t time = (rows * cols + 255) / 256 * kTiles[f].round;
        if (time >= best || !fits(f)) continue;
        best = time;
        n.form = f;
        n.tilesM = rows;
        n.tilesN = cols;
        // A ring of 128 x 128 fits LDS once with six steps, twice with four: 512 x 8192
        // 28.9 and 32.8, 2048 x 4096, two rounds, 54.1 and 50.5.
        n.stages = f == kTile64 ? 8 : f == kTile128x64 || (f == kTile128 && rows * cols <= 256) ? 6 : 4;
    }
    // Ranges of k of 1024 bytes and more where the tiles leave units idle, from
    // k = 4096 on: 64 x 4096 of 2048 takes 9.2 whole and 10.7 in two, of 4096 14.5 and,
    // in four, 11.3, 64 x 2048 of 8192 24.1 and, in eight, 12.3.
    if (room && p->k >= 4096) n.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({256 / (n.tilesM * n.tilesN), p->k / 1024, 32})));
    return n;
}

/// The plan a launch has the workspace for.
Plan planFor(const mlkd_matmul_i8* p) {
    const int64_t need = mlkd_matmul_i8_work_bytes(p);
    return planOf(p, need == 0 || (p->work != nullptr && p->work_bytes >= need));
}

template <typename T, int MB>
void launchFew(const mlkd_matmul_i8* p, const Plan& n, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((p->n + 16 * n.nb - 1) / (16 * n.nb), int64_t{1} << 20));
    auto* kernel = n.aligned ? (n.nb == 2 ? matmulI8Few<T, MB, 2, true> : matmulI8Few<T, MB, 1, true>)
                             : (n.nb == 2 ? matmulI8Few<T, MB, 2, false> : matmulI8Few<T, MB, 1, false>);
    constexpr int64_t kRows = (int64_t{16} * MB) << 15;   // a launch's: blocks of them along y
    for (int64_t r = 0; r < p->m; r += kRows) {
        mlkd_matmul_i8 part = *p;
        part.a += r * p->lda;
        part.a_scale += r;
        part.out = static_cast<T*>(p->out) + r * p->ldo;
        part.m = std::min(kRows, p->m - r);
        hipLaunchKernelGGL(kernel, dim3(grid, static_cast<unsigned>((part.m + 16 * MB - 1) / (16 * MB))), dim3(512), 0, st, part, n.wide ? 1 : 0);
    }
}

template <typename T, int WM, int WN, int MT, int NT, int kStages>
int launchTiles(const TileArgs& a, hipStream_t st) {
    constexpr int bytes = (WM * MT + WN * NT) * 16 * kStep * kStages;
    auto* kernel = matmulI8Tiles<T, WM, WN, MT, NT, kStages>;
    // Once per process; a function-local static initializes thread-safely.
    static const bool allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                    bytes) == hipSuccess;
    if (!allowed) return MLKD_RT_LAUNCH;
    const int64_t grid = static_cast<int64_t>(a.tilesM) * a.tilesN * a.splits;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(WM * WN * 64), bytes, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

template <typename T>
int launch(const mlkd_matmul_i8* p, hipStream_t st) {
    const Plan n = planFor(p);
    if (n.form == kFew) {
        n.mb == 1 ? launchFew<T, 1>(p, n, st) : n.mb == 2 ? launchFew<T, 2>(p, n, st) : launchFew<T, 4>(p, n, st);
        return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
    }
    TileArgs a{*p, static_cast<int>(n.tilesM), static_cast<int>(n.tilesN), n.splits, n.wide ? 1 : 0, nullptr, (p->n + 3) / 4 * 4};
    if (n.splits > 1) a.work = reinterpret_cast<int*>(static_cast<char*>(p->work) + packBytes(p, n));
    if (n.pack) {
        int8_t* to = static_cast<int8_t*>(p->work);
        const int64_t pitch = pitchOf(p), pieces = (p->m + p->n) * pitch / 16;
        hipLaunchKernelGGL(matmulI8Pack, dim3(static_cast<unsigned>(std::min<int64_t>((pieces + 255) / 256, int64_t{1} << 16))), dim3(256), 0, st, *p, to, pitch);
        if (hipGetLastError() != hipSuccess) return MLKD_RT_LAUNCH;
        a.p.a = to;
        a.p.b = to + p->m * pitch;
        a.p.lda = a.p.ldb = a.p.k = pitch;
    }
    const int rc = n.form == kTile256      ? launchTiles<T, 4, 2, 4, 8, 4>(a, st)
                   : n.form == kTile128    ? n.stages == 6 ? launchTiles<T, 2, 2, 4, 4, 6>(a, st) : launchTiles<T, 2, 2, 4, 4, 4>(a, st)
                   : n.form == kTile128x64 ? launchTiles<T, 2, 2, 4, 2, 6>(a, st)
                                           : launchTiles<T, 2, 2, 2, 2, 8>(a, st);
    if (rc != 0 || n.splits == 1) return rc;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p->m * a.ldw / 4 + 255) / 256, int64_t{1} << 16)));
    hipLaunchKernelGGL(matmulI8Join<T>, grid, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

int64_t mlkd_matmul_i8_work_bytes(const mlkd_matmul_i8* p) {
    const Plan n = planOf(p, true);
    return packBytes(p, n) + sumBytes(p, n);
}

const char* mlkd_matmul_i8_kernel_names(const mlkd_matmul_i8* p) {
    static thread_local std::string name;
    const std::string type = typeName(p->dtype);
    const Plan n = planFor(p);
    if (n.form == kFew) {
        name = "matmulI8Few<" + type + ", " + std::to_string(n.mb) + ", " + std::to_string(n.nb) + (n.aligned ? ", true>" : ", false>");
        return name.c_str();
    }
    name = std::string(n.pack ? "matmulI8Pack+" : "") + "matmulI8Tiles<" + type +
           (n.form == kTile256 ? ", 4, 2, 4, 8, " : n.form == kTile128 ? ", 2, 2, 4, 4, " : n.form == kTile128x64 ? ", 2, 2, 4, 2, " : ", 2, 2, 2, 2, ") +
           std::to_string(n.stages) + ">";
    if (n.splits > 1) name += "+matmulI8Join<" + type + ">";
    return name.c_str();
}

int mlkd_launch_matmul_i8(const mlkd_matmul_i8* p, void* stream) {
    if (p->m == 0) return 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return p->dtype == MLKD_F32 ? launch<float>(p, st) : p->dtype == MLKD_F16 ? launch<_Float16>(p, st) : launch<__bf16>(p, st);
}

}  // extern "C"
