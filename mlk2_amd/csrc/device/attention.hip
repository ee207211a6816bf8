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
            for (int32_t j0 = 0; j0 < n; j0 += 64) {
                const int seen = min(64, n - j0);
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
/// 2^(m_i - m), m the largest maximum. LPR lanes a row, 4 columns each.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void attentionJoin(mlk::TileArgs a) {
    const mlkd_attention& p = a.p;
    using mlk::f32x4;
    const int ln = threadIdx.x % LPR;
    const int64_t rows = p.q_rows * p.heads;
    for (int64_t r = blockIdx.x * int64_t{256 / LPR} + threadIdx.x / LPR; r < rows; r += static_cast<int64_t>(gridDim.x) * (256 / LPR)) {
        const int64_t t = r / p.heads;
        if (sequenceOf(p, t) < 0) continue;
        float m = mlk::kLowest;
        for (int i = 0; i < a.parts; ++i) m = fmaxf(m, a.ml[i * rows + r].x);
        float l = 0.0f;
        f32x4 sum = {};
        for (int i = 0; i < a.parts; ++i) {
            const float2 ml = a.ml[i * rows + r];
            if (ml.y == 0.0f) continue;   // no weights: its sums may not have been written
            const float w = __builtin_amdgcn_exp2f(ml.x - m);
            l += ml.y * w;
            if (4 * ln < p.dim) sum += w * *reinterpret_cast<const f32x4*>(a.acc + (i * rows + r) * p.dim + 4 * ln);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (4 * ln < p.dim) {
            mlk::Vec4<T> v;
#pragma unroll
            for (int f = 0; f < 4; ++f) v[f] = static_cast<T>(sum[f] * inv);
            *reinterpret_cast<mlk::Vec4<T>*>(static_cast<T*>(p.out) + t * p.out_stride + (r % p.heads) * p.dim + 4 * ln) = v;
        }
        if (p.lse != nullptr && ln == 0) p.lse[r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

/// How a launch runs: on the matrix cores or row by row, with which row
/// blocks, in how many key ranges.
struct Plan {
    bool tiles{false};
    bool shared{false};     // the prefix for all sequences' rows together
    int wavesOwn{0}, wavesPrefix{0};   // of a row block, 32 rows each
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
    if (p->q_rows * (p->heads / p->kv_heads) >= (int64_t{1} << 30)) return false;   // rows are counted in 32 bits
    return aligned(p->q, p->q_stride, 16, size) && aligned(p->k, p->k_stride, 16, size) && aligned(p->v, p->v_stride, 16, size) &&
           aligned(p->out, p->out_stride, 4 * size, size) && aligned(p->prefix_k, p->prefix_k_stride, 16, size) &&
           aligned(p->prefix_v, p->prefix_v_stride, 16, size);
}

/// Tiles of the matrix-core kernels: keys a tile and tiles in LDS.
constexpr int keysOf(int size, int dt, int waves) { return waves > 1 && size == 2 && dt <= 128 ? 64 : 32; }
constexpr int stagesOf(int size, int dt, int waves) {
    const int bytes = 2 * keysOf(size, dt, waves) * (dt <= 64 ? 64 : dt <= 128 ? 128 : 256) * size;   // of a tile
    return waves > 1 ? (bytes <= 32768 ? 4 : 2) : bytes <= 16384 ? 4 : 2;
}
constexpr int wideOf(int size, int dt) { return size == 2 && dt <= 128 ? 8 : 4; }
int dimOf(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }

Plan planOf(const mlkd_attention* p) {
    Plan n;
    n.tiles = tilesApply(p);
    if (!n.tiles) return n;
    const int64_t group = p->heads / p->kv_heads;
    const int64_t each = (p->q_rows + p->sequences - 1) / p->sequences * group;   // rows of a sequence, on average
    const int64_t keys = std::max<int64_t>(1, p->kv_rows / p->sequences);
    const int wide = wideOf(p->dtype == MLKD_F32 ? 4 : 2, dimOf(p->dim));
    n.wavesOwn = each > 64 ? wide : 1;
    n.shared = p->prefix_k != nullptr && n.wavesOwn == 1;
    auto ranges = [&](int64_t blocks, int64_t count, int64_t fill) {
        return static_cast<int>(std::max<int64_t>(1, std::min({fill / std::max<int64_t>(1, blocks * p->kv_heads), count / 128, int64_t{64}})));
    };
    if (n.wavesOwn == 1) n.splitsOwn = ranges((p->q_rows * group + 31) / 32 + p->sequences - 1, keys, 1024);
    if (n.shared) {
        n.wavesPrefix = wide;
        n.splitsPrefix = ranges((p->q_rows * group + 32 * wide - 1) / (32 * wide), p->prefix_rows, 256);
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

template <typename T, int DT, int NW>
int launchTiles(const mlk::TileArgs& a, int64_t blocks, hipStream_t st) {
    constexpr int KEYS = keysOf(sizeof(T), DT, NW), STAGES = stagesOf(sizeof(T), DT, NW);
    constexpr int bytes = mlk::Tiles<T, DT, NW, KEYS, STAGES>::kLds;
    auto* kernel = mlk::attentionTiles<T, DT, NW, KEYS, STAGES>;
    // Once per process; a function-local static initializes thread-safely.
    static const bool allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                    bytes) == hipSuccess;
    if (!allowed) return MLKD_RT_LAUNCH;
    const int64_t grid = blocks * a.splits * a.p.kv_heads;
    if (grid * NW * 64 >= (int64_t{1} << 32)) return -1;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(NW * 64), bytes, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

/// The row blocks of a launch: at most so many for any lengths.
int64_t rowBlocks(const mlk::TileArgs& a, int waves) {
    const int64_t rows = a.p.q_rows * (a.p.heads / a.p.kv_heads), each = 32 * waves;
    return a.all_rows != 0 ? (rows + each - 1) / each : rows / each + std::min<int64_t>(a.p.sequences, rows);
}

template <typename T, int DT>
int launchWaves(const mlk::TileArgs& a, int waves, hipStream_t st) {
    constexpr int WIDE = wideOf(sizeof(T), DT);
    return waves == 1 ? launchTiles<T, DT, 1>(a, rowBlocks(a, 1), st) : launchTiles<T, DT, WIDE>(a, rowBlocks(a, WIDE), st);
}

template <typename T>
int launchDim(const mlk::TileArgs& a, int waves, hipStream_t st) {
    switch (dimOf(a.p.dim)) {
        case 64: return launchWaves<T, 64>(a, waves, st);
        case 96: return launchWaves<T, 96>(a, waves, st);
        case 128: return launchWaves<T, 128>(a, waves, st);
        default: return launchWaves<T, 256>(a, waves, st);
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
        if (const int rc = launchDim<T>(a, n.wavesPrefix, st); rc != 0) return rc;
        a.part0 = n.splitsPrefix;
        a.all_rows = 0;
    }
    a.keys = n.shared ? 2 : 3;
    a.splits = n.splitsOwn;
    if (const int rc = launchDim<T>(a, n.wavesOwn, st); rc != 0) return rc;
    if (a.parts == 0) return 0;
    const int64_t rows = p->q_rows * p->heads;
    auto* join = p->dim <= 64 ? attentionJoin<T, 16> : p->dim <= 128 ? attentionJoin<T, 32> : attentionJoin<T, 64>;
    const int per = p->dim <= 64 ? 16 : p->dim <= 128 ? 8 : 4;
    hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(std::min<int64_t>((rows + per - 1) / per, int64_t{1} << 20))), dim3(256), 0, st, a);
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
    auto tiles = [&](int waves) {
        return "attentionTiles<" + type + ", " + std::to_string(dt) + ", " + std::to_string(waves) + ", " +
               std::to_string(keysOf(size, dt, waves)) + ", " + std::to_string(stagesOf(size, dt, waves)) + ">";
    };
    name = n.shared ? tiles(n.wavesPrefix) + "+" + tiles(n.wavesOwn) : tiles(n.wavesOwn);
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
