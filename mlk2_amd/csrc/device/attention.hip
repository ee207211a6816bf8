// Attention over packed sequences, out = softmax(scale q k^T) v, with grouped
// heads, causal or not, keys in a cache, and optionally behind a prefix that
// all sequences share.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <string>

#include "attention_tiles.h"
#include "runtime_abi.h"

namespace {

using mlk::prefixOf;
using mlk::SeqSpan;
using mlk::spanOf;

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float waveMax(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

__device__ __forceinline__ float waveSum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ float lane(float v, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}

/// The sequence that holds query row t, or -1: the last whose first row is at
/// or before it, where that one reaches it.
__device__ __forceinline__ int sequenceOf(const mlkd_attention& p, int64_t t) {
    int lo = 0, hi = p.sequences;   // q_offsets[lo - 1] <= t < q_offsets[hi], as far as they are in order
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.q_offsets[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && t < p.q_offsets[lo] ? lo - 1 : -1;
}

/// A query row in one wave, with any strides and alignment: a lane per key for
/// the scores (f32 sums over d), then a lane per output column. The running
/// maximum and sum take one pass over the keys; only keys that the row sees
/// are read.
template <typename T>
__global__ __launch_bounds__(256) void attentionRows(mlkd_attention p) {
    const int ln = threadIdx.x & 63, d = p.dim, group = p.heads / p.kv_heads;
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4, rows = p.q_rows * p.heads;
    const float scale = static_cast<float>(p.scale * 1.4426950408889634);
    const int32_t np = prefixOf(p);
    for (int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); r < rows; r += waves) {
        const int64_t t = r / p.heads;
        const int h = static_cast<int>(r % p.heads), g = h / group;
        const int b = sequenceOf(p, t);
        if (b < 0) continue;
        const SeqSpan s = spanOf(p, b);
        const int32_t own = p.causal != 0
                                ? static_cast<int32_t>(max(int64_t{0}, min(int64_t{s.nk}, t - s.q0 + 1 + s.nk - s.nq)))
                                : s.nk;
        const T* qr = static_cast<const T*>(p.q) + t * p.q_stride + static_cast<int64_t>(h) * d;
        float q[4], acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = ln + 64 * i < d ? static_cast<float>(qr[ln + 64 * i]) * scale : 0.0f;
            acc[i] = 0.0f;
        }
        float m = -INFINITY, l = 0.0f;
        for (int part = 0; part < 2; ++part) {
            const int32_t n = part == 0 ? np : own;
            const int64_t ks = part == 0 ? p.prefix_k_stride : p.k_stride, vs = part == 0 ? p.prefix_v_stride : p.v_stride;
            const T* k = static_cast<const T*>(part == 0 ? p.prefix_k : p.k) + (part == 0 ? 0 : s.k0 * ks) + g * d;
            const T* v = static_cast<const T*>(part == 0 ? p.prefix_v : p.v) + (part == 0 ? 0 : s.k0 * vs) + g * d;
            for (int64_t j0 = 0; j0 < n; j0 += 64) {
                const int seen = static_cast<int>(min(int64_t{64}, n - j0));
                const T* kr = k + (j0 + min(ln, seen - 1)) * ks;
                float x = 0.0f;
                for (int c = 0; c < d; ++c) x += lane(c < 64 ? q[0] : c < 128 ? q[1] : c < 192 ? q[2] : q[3], c & 63) * static_cast<float>(kr[c]);
                if (ln >= seen) x = -INFINITY;
                const float top = fmaxf(m, waveMax(x));
                const float base = top == -INFINITY ? 0.0f : top;
                const float w = __builtin_amdgcn_exp2f(x - base), keep = __builtin_amdgcn_exp2f(m - base);
                l = l * keep + waveSum(w);
                m = top;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] *= keep;
                for (int j = 0; j < seen; ++j) {
                    const float wj = lane(w, j);
                    const T* vr = v + (j0 + j) * vs;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (ln + 64 * i < d) acc[i] += wj * static_cast<float>(vr[ln + 64 * i]);
                    }
                }
            }
        }
        // A sum of no weights; one that is NaN stays one.
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* o = static_cast<T*>(p.out) + t * p.out_stride + static_cast<int64_t>(h) * d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ln + 64 * i < d) o[ln + 64 * i] = static_cast<T>(acc[i] * inv);
        }
        if (p.lse != nullptr && ln == 0) p.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

/// The results of key ranges joined: out = sum acc_i 2^(m_i - m) / sum l_i
/// 2^(m_i - m), m the largest maximum. A wave a row, LPR lanes to a range with 4
/// columns each, so that ranges are read side by side, four of them in flight.
/// Bound by the waits of a row's few dependent reads: 2048 rows of 128 columns
/// and 17 ranges in 6.7 us (18 MB), 11688 rows of 64 and 5 ranges in 9.3.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void attentionJoin(mlk::TileArgs a) {
    const mlkd_attention& p = a.p;
    using mlk::f32x4;
    constexpr int SIDE = 64 / LPR;
    const int ln = threadIdx.x & 63, column = ln % LPR * 4;
    const int64_t rows = p.q_rows * p.heads;
    for (int64_t r = blockIdx.x * int64_t{4} + threadIdx.x / 64; r < rows; r += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t t = rows < (int64_t{1} << 30) ? static_cast<int>(r) / a.by_heads : r / p.heads;
        // A row of no sequence is left alone.
        bool held = false;
        for (int s = ln; s < p.sequences; s += 64) held |= p.q_offsets[s] <= t && t < p.q_offsets[s + 1];
        // The weights of the ranges, lane i those of i and 64 + i; below 0: a
        // range without keys, its sums may not have been written.
        float2 ml[2];
        float w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) ml[h] = ln + 64 * h < a.parts ? a.ml[(ln + 64 * h) * rows + r] : make_float2(mlk::kLowest, 0.0f);
        if (!__any(held)) continue;
        const float m = waveMax(fmaxf(ml[0].x, ml[1].x));
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = __builtin_amdgcn_exp2f(ml[h].x - m);
        const float l = waveSum(ml[0].y * w[0] + ml[1].y * w[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = ml[h].y == 0.0f ? -1.0f : w[h];
        f32x4 sum = {};
        const float* from = a.acc + r * p.dim + column;
#pragma unroll 1
        for (int i0 = 0; i0 < a.parts; i0 += 4 * SIDE) {
            f32x4 v[4];
            float u[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = i0 + n * SIDE + ln / LPR;
                u[n] = __shfl(i0 + n * SIDE < 64 ? w[0] : w[1], i & 63);
                v[n] = f32x4{};
                if (i < a.parts && u[n] >= 0.0f && column < p.dim) v[n] = *reinterpret_cast<const f32x4*>(from + i * rows * p.dim);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) sum += fmaxf(u[n], 0.0f) * v[n];
        }
#pragma unroll
        for (int d = LPR; d < 64; d *= 2) {
#pragma unroll
            for (int f = 0; f < 4; ++f) sum[f] += __shfl_xor(sum[f], d);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (column < p.dim && ln < LPR) {
            mlk::Vec4<T> v;
#pragma unroll
            for (int f = 0; f < 4; ++f) v[f] = static_cast<T>(sum[f] * inv);
            *reinterpret_cast<mlk::Vec4<T>*>(static_cast<T*>(p.out) + t * p.out_stride + (r % p.heads) * p.dim + column) = v;
        }
        if (p.lse != nullptr && ln == 0) p.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

/// Row blocks of the matrix-core kernels: one wave of 32 rows; eight waves in
/// two groups, 128 rows; the widest, see wavesOf.
enum Block { kNarrow, kHalves, kWide };

/// How a launch runs: on the matrix cores or row by row, with which row
/// blocks, in how many key ranges.
struct Plan {
    bool tiles{false};
    bool shared{false};     // the prefix for all sequences' rows together
    Block own{kNarrow}, prefix{kNarrow};
    int splitsOwn{1}, splitsPrefix{0};
    int parts() const { return splitsOwn + splitsPrefix > 1 ? splitsOwn + splitsPrefix : 0; }
};

bool aligned(const void* ptr, int64_t stride, int bytes, int size) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && stride * size % bytes == 0 && stride < (int64_t{1} << 22);
}

/// The matrix-core kernels take rows whose 16-byte pieces are aligned.
bool tilesApply(const mlkd_attention* p) {
    const int size = p->dtype == MLKD_F32 ? 4 : 2;
    if (p->dim % 8 != 0) return false;
    // A block finds its sequence by reading the lengths 64 at a time from the
    // batch's end: 64 dependent rounds at most, then by halving, row by row.
    if (p->sequences > 4096) return false;
    // Rows and keys, with a tile's more, are counted in 32 bits.
    if (p->q_rows * (p->heads / p->kv_heads) >= (int64_t{1} << 30) || std::max(p->kv_rows, p->prefix_rows) > (int64_t{1} << 30)) return false;
    return aligned(p->q, p->q_stride, 16, size) && aligned(p->k, p->k_stride, 16, size) && aligned(p->v, p->v_stride, 16, size) &&
           aligned(p->out, p->out_stride, 16, size) && aligned(p->prefix_k, p->prefix_k_stride, 16, size) &&
           aligned(p->prefix_v, p->prefix_v_stride, 16, size);
}

/// The matrix-core kernels: waves of a row block and their groups, keys of a
/// tile, tiles in LDS.
constexpr bool eight(int size, int dt) { return size == 2 && dt <= 128; }
constexpr int wavesOf(Block block, int size, int dt) { return block == kNarrow ? 1 : eight(size, dt) ? 8 : 4; }
constexpr int groupsOf(Block block) { return block == kHalves ? 2 : 1; }
constexpr int keysOf(Block block, int size, int dt) { return wavesOf(block, size, dt) == 8 ? 64 : 32; }
constexpr int stagesOf(Block block, int size, int dt) {
    const int bytes = 2 * keysOf(block, size, dt) * (dt <= 64 ? 64 : dt <= 128 ? 128 : 256) * size;   // of a tile
    return block != kNarrow ? (bytes <= 32768 ? 4 : 2) : size == 2 && bytes <= 16384 ? 4 : 2;
}
constexpr int rowsOf(Block block, int size, int dt) { return 32 * wavesOf(block, size, dt) / groupsOf(block); }
int dimOf(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }

Plan planOf(const mlkd_attention* p) {
    Plan n;
    n.tiles = tilesApply(p);
    if (!n.tiles) return n;
    const int64_t group = p->heads / p->kv_heads;
    const int64_t tokens = (p->q_rows + p->sequences - 1) / p->sequences, each = tokens * group;   // rows of a sequence, on average
    const int64_t keys = std::max<int64_t>(1, p->kv_rows / p->sequences), all = keys + (p->prefix_k != nullptr ? p->prefix_rows : 0);
    const int size = p->dtype == MLKD_F32 ? 4 : 2, dt = dimOf(p->dim);
    // Row blocks of all sequences' and all key/value heads', of rows of average sequences.
    auto blocks = [&](int64_t count, int64_t rows, Block block) {
        const int64_t of = rowsOf(block, size, dt);
        return count * ((rows + of - 1) / of) * p->kv_heads;
    };
    auto ranges = [&](int64_t count, int64_t keys, int64_t fill) {
        return static_cast<int>(std::max<int64_t>(1, std::min({fill / std::max<int64_t>(1, count), keys / 128, int64_t{64}})));
    };
    const int64_t narrow = blocks(p->sequences, each, kNarrow), wide = blocks(p->sequences, each, kWide);
    // One wave to a block where a sequence has two blocks' rows at most, and, of
    // 16-bit types, where there is little to do: 19 tokens over 1000 keys, 32 and
    // 8 heads of 128, in 15 us against 26, 256 over 256 in 17 against 13.5.
    const bool few = each <= 64 || (size == 2 && narrow * all <= 32768);
    // Half the rows to a workgroup where whole blocks leave compute units idle:
    // 1024 tokens, every key seen, in 29 us against 39, 1536 in 68 against 55.
    // Where the rows see unlike numbers of keys, the shorter blocks also even
    // out what the units do: 2048 tokens in 55 us against 57, 2304 in 75
    // against 80, 4096 in 183 against 161.
    const bool level = p->causal == 0 || all >= 2 * tokens;
    if (few) n.own = kNarrow;
    else if (eight(size, dt)) n.own = wide <= (level ? 128 : 320) ? kHalves : kWide;
    // f32 takes its time in the products alone, 16 times those of 16 bits: one
    // wave to a block and key ranges where blocks of four leave units idle (two
    // sequences of 1001, 8 heads of 64: 51 us against 79; four, 16 heads: 182
    // against 143).
    else n.own = size == 4 && wide < 256 ? kNarrow : kWide;
    n.shared = p->prefix_k != nullptr && each <= 64;
    // Ranges of 128 keys and more, so many that each SIMD has a wave (f32, with
    // two tiles in LDS: two).
    const int64_t count = blocks(p->sequences, each, n.own);
    if (n.own == kNarrow) n.splitsOwn = ranges(narrow, n.shared ? keys : all, size == 4 ? 2048 : 1024);
    // Ranges of 256 keys and more for larger blocks that leave half the units
    // idle, where the keys make up for the join: two sequences of 100 tokens
    // over 8192 keys, 32 and 8 heads of 128, in 55 us against 149, 8 of 19 over
    // 2000 in 30 against 45; one of 512 over 512, 16 and 4 heads, in 24 against 18.
    else if (count <= 128 && all >= 768) n.splitsOwn = ranges(count, all / 2, 256);
    if (n.shared) {
        const int64_t rows = p->q_rows * group;
        n.prefix = eight(size, dt) && blocks(1, rows, kWide) <= 128 ? kHalves : kWide;
        n.splitsPrefix = ranges(blocks(1, rows, n.prefix), p->prefix_rows, 256);
    }
    return n;
}

/// The plan a launch has the workspace for.
Plan planFor(const mlkd_attention* p) {
    Plan n = planOf(p);
    if (n.parts() > 0 && (p->work == nullptr || p->work_bytes < mlkd_attention_work_bytes(p))) {
        n.shared = false;
        n.splitsOwn = 1;
        n.splitsPrefix = 0;
    }
    return n;
}

mlk::Divider dividerOf(int d) {
    if (d == 1) return {0, 0};
    int up = 0;
    while ((int64_t{1} << up) < d) ++up;
    return {static_cast<uint32_t>(((uint64_t{1} << (31 + up)) + d - 1) / d), up - 1};
}

/// The row blocks of a launch: at most so many for any lengths.
int64_t rowBlocks(const mlk::TileArgs& a, int each) {
    const int64_t rows = a.p.q_rows * (a.p.heads / a.p.kv_heads);
    return a.all_rows != 0 ? (rows + each - 1) / each : rows / each + std::min<int64_t>(a.p.sequences, rows);
}

template <typename T, int DT, Block BLOCK>
int launchTiles(mlk::TileArgs a, hipStream_t st) {
    a.by_group = dividerOf(a.p.heads / a.p.kv_heads);
    a.by_kv_heads = dividerOf(a.p.kv_heads);
    a.by_splits = dividerOf(a.splits);
    constexpr int NW = wavesOf(BLOCK, sizeof(T), DT), KG = groupsOf(BLOCK), KEYS = keysOf(BLOCK, sizeof(T), DT);
    constexpr int STAGES = stagesOf(BLOCK, sizeof(T), DT), bytes = mlk::Tiles<T, DT, NW, KG, KEYS, STAGES>::kLds;
    auto* kernel = mlk::attentionTiles<T, DT, NW, KG, KEYS, STAGES>;
    // Once per process; a function-local static initializes thread-safely.
    static const bool allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                    bytes) == hipSuccess;
    if (!allowed) return MLKD_RT_LAUNCH;
    const int64_t grid = rowBlocks(a, rowsOf(BLOCK, sizeof(T), DT)) * a.splits * a.p.kv_heads;
    if (grid * NW * 64 >= (int64_t{1} << 32)) return -1;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(NW * 64), bytes, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

template <typename T, int DT>
int launchBlock(const mlk::TileArgs& a, Block block, hipStream_t st) {
    if constexpr (eight(sizeof(T), DT)) {
        if (block == kHalves) return launchTiles<T, DT, kHalves>(a, st);
    }
    return block == kNarrow ? launchTiles<T, DT, kNarrow>(a, st) : launchTiles<T, DT, kWide>(a, st);
}

template <typename T>
int launchDim(const mlk::TileArgs& a, Block block, hipStream_t st) {
    switch (dimOf(a.p.dim)) {
        case 64: return launchBlock<T, 64>(a, block, st);
        case 96: return launchBlock<T, 96>(a, block, st);
        case 128: return launchBlock<T, 128>(a, block, st);
        default: return launchBlock<T, 256>(a, block, st);
    }
}

template <typename T>
int launchPlan(const mlkd_attention* p, const Plan& n, hipStream_t st) {
    mlk::TileArgs a{};
    a.p = *p;
    a.parts = n.parts();
    if (a.parts > 0) {
        a.acc = static_cast<float*>(p->work);
        a.ml = reinterpret_cast<float2*>(a.acc + a.parts * p->q_rows * p->heads * p->dim);
    }
    if (n.shared) {
        a.keys = 1;
        a.all_rows = 1;
        a.splits = n.splitsPrefix;
        if (const int rc = launchDim<T>(a, n.prefix, st); rc != 0) return rc;
        a.part0 = n.splitsPrefix;
        a.all_rows = 0;
    }
    a.keys = n.shared ? 2 : 3;
    a.splits = n.splitsOwn;
    if (const int rc = launchDim<T>(a, n.own, st); rc != 0) return rc;
    if (a.parts == 0) return 0;
    a.by_heads = dividerOf(p->heads);
    const int64_t rows = p->q_rows * p->heads;
    auto* join = p->dim <= 64 ? attentionJoin<T, 16> : p->dim <= 128 ? attentionJoin<T, 32> : attentionJoin<T, 64>;
    hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20))), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

int64_t mlkd_attention_work_bytes(const mlkd_attention* p) {
    return planOf(p).parts() * p->q_rows * p->heads * (p->dim * static_cast<int64_t>(sizeof(float)) + static_cast<int64_t>(sizeof(float2)));
}

const char* mlkd_attention_kernel_names(const mlkd_attention* p) {
    static thread_local std::string name;
    const std::string type = typeName(p->dtype);
    const Plan n = planFor(p);
    if (!n.tiles) {
        name = "attentionRows<" + type + ">";
        return name.c_str();
    }
    const int dt = dimOf(p->dim), size = p->dtype == MLKD_F32 ? 4 : 2;
    auto tiles = [&](Block block) {
        std::string s = "attentionTiles<" + type;
        for (const int v : {dt, wavesOf(block, size, dt), groupsOf(block), keysOf(block, size, dt), stagesOf(block, size, dt)}) s += ", " + std::to_string(v);
        return s + ">";
    };
    name = n.shared ? tiles(n.prefix) + "+" + tiles(n.own) : tiles(n.own);
    if (n.parts() > 0) name += "+attentionJoin<" + type + ", " + std::to_string(dt <= 64 ? 16 : dt <= 128 ? 32 : 64) + ">";
    return name.c_str();
}

int mlkd_launch_attention(const mlkd_attention* p, void* stream) {
    const int64_t rows = p->q_rows * p->heads;
    if (rows == 0) return 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (const Plan n = planFor(p); n.tiles) {
        const int rc = p->dtype == MLKD_F32   ? launchPlan<float>(p, n, st)
                       : p->dtype == MLKD_F16 ? launchPlan<_Float16>(p, n, st)
                                              : launchPlan<__bf16>(p, n, st);
        if (rc >= 0) return rc;   // else a grid past the limit
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->dtype == MLKD_F32 ? attentionRows<float> : p->dtype == MLKD_F16 ? attentionRows<_Float16> : attentionRows<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, *p);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
