// Attention over packed sequences whose keys and values are a cache's in 4 bits.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "attention_kv4_tiles.h"
#include "attention_rows.h"
#include "bits.h"
#include "runtime_abi.h"

namespace {

using mlk::SeqSpan;
using mlk::spanOf;

/// A query row in one wave, with any even dim, strides and alignment: a lane per
/// key for the scores, then a lane per output column. 32 single tokens over 1000 to
/// 8192 keys of dim 120 take 5.3 ms, 2048 tokens 8.8.
template <typename T>
__global__ __launch_bounds__(256) void attentionKv4Rows(mlk::Kv4Args args) {
    const mlkd_attention& p = args.t.p;
    const int ln = threadIdx.x & 63, d = p.dim, group = p.heads / p.kv_heads;
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4, rows = p.q_rows * p.heads;
    for (int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6); r < rows; r += waves) {
        const int64_t t = r / p.heads;
        const int h = static_cast<int>(r % p.heads), g = h / group;
        const int b = sequenceOf(p, t);
        if (b < 0) continue;
        const SeqSpan s = spanOf(p, b);
        const int64_t own = p.causal != 0 ? max(int64_t{0}, min(int64_t{s.nk}, t - s.q0 + 1 + s.nk - s.nq)) : s.nk;
        const T* qr = static_cast<const T*>(p.q) + t * p.q_stride + static_cast<int64_t>(h) * d;
        float q[4], acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = ln + 64 * i < d ? static_cast<float>(qr[ln + 64 * i]) : 0.0f;
            acc[i] = 0.0f;
        }
        // A row's elements are taken at a size below 1, so that sums of them times codes
        // stay in range, and 2^lacks comes with the key's scale.
        const float size = waveMax(fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3]))));
        const int by = size < INFINITY ? __builtin_amdgcn_frexp_expf(size) : 0, lacks = by + args.up + __builtin_amdgcn_frexp_expf(args.codes) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = __builtin_amdgcn_ldexpf(q[i], -by);
        auto query = [&](int c) { return lane(c < 64 ? q[0] : c < 128 ? q[1] : c < 192 ? q[2] : q[3], c & 63); };
        float m = -INFINITY, l = 0.0f;
        const uint8_t* k = static_cast<const uint8_t*>(p.k) + s.k0 * p.k_stride + g * (d / 2);
        const uint8_t* v = static_cast<const uint8_t*>(p.v) + s.k0 * p.v_stride + g * (d / 2);
        for (int64_t j0 = 0; j0 < own; j0 += 64) {
            const int seen = static_cast<int>(min(int64_t{64}, own - j0));
            const int64_t j = j0 + min(ln, seen - 1), at = (s.k0 + j) * p.kv_heads + g;
            const uint8_t* kr = k + j * p.k_stride;
            float x = 0.0f;
            for (int c = 0; c < d / 2; ++c) {
                const mlk::F32x2 n = mlk::numbersOf<0>(kr[c]);
                x += query(2 * c) * n[0];
                x += query(2 * c + 1) * n[1];
            }
            const float ks = args.k_scale[at];
            x = __builtin_amdgcn_ldexpf(x * (__builtin_amdgcn_frexp_mantf(ks) * args.c), __builtin_amdgcn_frexp_expf(ks) + lacks);
            const float vs = args.v_scale[at];
            if (ln >= seen) x = -INFINITY;
            const float top = fmaxf(m, waveMax(x));
            const float base = top == -INFINITY ? 0.0f : top;
            const float w = __builtin_amdgcn_exp2f(x - base), keep = __builtin_amdgcn_exp2f(m - base);
            l = l * keep + waveSum(w);
            m = top;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= keep;
            for (int i = 0; i < seen; ++i) {
                const float wi = lane(w, i) * lane(vs, i);
                const uint8_t* vr = v + (j0 + i) * p.v_stride;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int c = ln + 64 * n;
                    if (c < d) acc[n] += wi * mlk::numbersOf<0>(vr[c >> 1] >> (c & 1) * 4)[0];
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

/// How a launch runs: on the matrix cores or row by row, rows of a block, waves to
/// one, units of a head that the keys are dealt out to in so many ranges at most (0:
/// one range to a row block).
struct Plan {
    bool tiles{false};
    int rows{16}, waves{4}, parts{0};
    int64_t units{0};
};

/// The matrix-core kernels take rows of q and out of whole 16-byte pieces, codes at 8
/// bytes, where their heads lie in any case, and heads of 32 and more elements in whole
/// sixteens. (Of 16 for codes as well, one kv head of dim 80 ran row by row.)
bool tilesApply(const mlkd_attention* p) {
    const int size = p->dtype == MLKD_F32 ? 4 : 2;
    // As attention's: a block reads the lengths 64 at a time, rows and keys are
    // counted in 32 bits.
    return p->dim % 16 == 0 && p->dim >= 32 && p->sequences <= 4096 && p->q_rows * (p->heads / p->kv_heads) < (int64_t{1} << 30) &&
           p->kv_rows <= (int64_t{1} << 30) && aligned(p->q, p->q_stride, 16, size) && aligned(p->out, p->out_stride, 16, size) &&
           aligned(p->k, p->k_stride, 8, 1) && aligned(p->v, p->v_stride, 8, 1);
}

int dimOf(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }
/// Row blocks of a launch: at most so many for any lengths.
int64_t rowBlocks(const mlkd_attention* p, int of) {
    const int64_t rows = p->q_rows * (p->heads / p->kv_heads);
    return rows / of + std::min<int64_t>(p->sequences, rows);
}

Plan planOf(const mlkd_attention* p) {
    Plan n;
    n.tiles = tilesApply(p);
    if (!n.tiles) return n;
    const int64_t group = p->heads / p->kv_heads, each = (p->q_rows + p->sequences - 1) / p->sequences * group;   // rows of a sequence, on average
    const int64_t keys = p->kv_rows / p->sequences;   // likewise
    // 64 sequences of 16 rows over 2048 keys, dim 128, bf16: 36.9 us by 16 and 45.8 by
    // 32 rows; of 20 rows 58.4 and 40.6.
    n.rows = each <= 16 ? 16 : 32;
    const int64_t blocks = p->sequences * ((each + n.rows - 1) / n.rows), most = rowBlocks(p, n.rows);
    // One wave a block needs no join of sums where there are blocks for all of them: 8 x
    // 2048 tokens 412 us, by four waves 489; 8 x 512 over 4096 keys 329 and 346; 4 x 125
    // to 1000 over up to 5000 242 and 204.
    n.waves = n.rows == 32 && blocks * p->kv_heads >= 4096 ? 1 : 4;
    n.units = most;
    // Dealt out by the keys, with a join, over the chip's room: three of four waves
    // of 16 rows a unit or two of 32. That costs 3 us for a sequence, 6 for 32 (more
    // row blocks, more parts to join), and a block's keys take 5.5 us a thousand, so it
    // pays where few blocks have many keys, or sequences unlike ones. Heads 32 on 8, dim
    // 128, bf16, from memory, us whole and dealt; sequences by their keys, all of one
    // length:
    //   1 by 1024 9.8 12.8, 1500 13.2 13.1, 2048 15.9 13.1, 8192 48.0 14.4
    //   8 by 1024 10.1 13.3, 2048 16.4 15.8, 4096 27.0 19.6, 8192 48.2 24.4
    //   16 by 2048 16.5 18.3, 4096 27.1 23.3, 8192 61.5 43.3
    //   32 by 2048 17.0 23.0, 4096 38.1 43.2, 8192 69.0 75.1, 16384 130 137
    //   48 by 8192 122 105; 64 by 4096 68.4 75.2
    // and of an eighth of that up to it:
    //   16 by 8192 48.6 27.0; 32 by 4096 28.0 26.4, 8192 60.9 51.7, 16384 117 92.6
    //   48 by 8192 102 74.1; 64 by 4096 55.5 55.3
    // The lengths are not known here, only the buffer's rows: 32 sequences are dealt from
    // 4500 rows each on, which costs equal ones 5 to 12 % and gains unlike ones 15 to 20,
    // 48 and 64 never. A cache with room takes the form of its rows (8 x 1000 keys in 8
    // x 8192 rows 12.7 for 10.2, 32 x 1000 in 32 x 8192 17.6 for 11.4), and sequences
    // that share rows have fewer each than they read (8 over the same 8192 48.2 whole,
    // 21.9 dealt). Prompts: 128 tokens over 1024 14.5 and 25.9, 4096 33.0 and 34.0, 8192
    // 57.1 and 43.2; twice 128 over 8192 59.6 and 67.0.
    const int64_t room = (n.rows == 16 ? 768 : 512) / p->kv_heads;
    if (p->sequences <= 64 && keys * (room - 2 * blocks) >= 1500 * room) {
        n.units = std::max(room, most + 1);
        n.parts = static_cast<int>(std::min<int64_t>(64, std::max<int64_t>(16, 4 * n.units / p->sequences)));
    }
    return n;
}

/// The plan a launch has the workspace for.
Plan planFor(const mlkd_attention_kv4* p) {
    Plan n = planOf(&p->a);
    if (n.parts > 0 && (p->a.work == nullptr || p->a.work_bytes < mlkd_attention_kv4_work_bytes(p))) {
        n.parts = 0;
        n.units = rowBlocks(&p->a, n.rows);
    }
    return n;
}

template <typename T, int DT, int ROWS, int NW>
int launchTiles(const mlk::Kv4Args& a, hipStream_t st) {
    constexpr int bytes = mlk::Kv4Tiles<T, DT, ROWS, NW>::kLds;
    auto* kernel = mlk::attentionKv4Tiles<T, DT, ROWS, NW>;
    // Once per process; a function-local static initializes thread-safely.
    static const bool allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                    bytes) == hipSuccess;
    if (!allowed) return MLKD_RT_LAUNCH;
    const int64_t grid = (static_cast<int64_t>(a.units) + 7) / 8 * 8 * a.t.p.kv_heads;
    if (grid * NW * 64 >= (int64_t{1} << 32)) return -1;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(NW * 64), bytes, st, a);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

template <typename T, int DT>
int launchForm(const mlk::Kv4Args& a, const Plan& n, hipStream_t st) {
    if (n.rows == 16) return launchTiles<T, DT, 16, 4>(a, st);
    if (n.waves == 4) return launchTiles<T, DT, 32, 4>(a, st);
    return launchTiles<T, DT, 32, 1>(a, st);
}

mlk::Kv4Args argsOf(const mlkd_attention_kv4* p) {
    mlk::Kv4Args a{};
    a.t.p = p->a;
    a.k_scale = p->k_scale;
    a.v_scale = p->v_scale;
    a.c = static_cast<float>(p->a.scale * 1.4426950408889634);
    const int all = std::fabs(a.c) >= 2.0f ? std::ilogb(a.c) : 0, codes = std::min(all, 13);
    a.c = std::ldexp(a.c, -all);
    a.codes = std::ldexp(1.0f, codes);
    a.up = all - codes;
    return a;
}

template <typename T>
int launchPlan(const mlkd_attention_kv4* p, const Plan& n, hipStream_t st) {
    mlk::Kv4Args a = argsOf(p);
    a.t.parts = n.parts;
    if (n.units >= (int64_t{1} << 30)) return -1;
    a.units = static_cast<int>(n.units);
    if (a.t.parts > 0) {
        a.t.acc = static_cast<float*>(p->a.work);
        a.t.ml = reinterpret_cast<float2*>(a.t.acc + a.t.parts * p->a.q_rows * p->a.heads * p->a.dim);
    }
    a.t.by_group = dividerOf(p->a.heads / p->a.kv_heads);
    a.t.by_kv_heads = dividerOf(p->a.kv_heads);
    a.t.by_heads = dividerOf(p->a.heads);
    int rc = 0;
    switch (dimOf(p->a.dim)) {
        case 64: rc = launchForm<T, 64>(a, n, st); break;
        case 96: rc = launchForm<T, 96>(a, n, st); break;
        case 128: rc = launchForm<T, 128>(a, n, st); break;
        default: rc = launchForm<T, 256>(a, n, st); break;
    }
    if (rc != 0 || a.t.parts == 0) return rc;
    const int64_t rows = p->a.q_rows * p->a.heads;
    auto* join = p->a.dim <= 64 ? attentionJoin<T, 16> : p->a.dim <= 128 ? attentionJoin<T, 32> : attentionJoin<T, 64>;
    hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20))), dim3(256), 0, st, a.t);
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

const char* typeName(int dtype) { return dtype == MLKD_F32 ? "float" : dtype == MLKD_F16 ? "_Float16" : "__bf16"; }

}  // namespace

extern "C" {

int64_t mlkd_attention_kv4_work_bytes(const mlkd_attention_kv4* p) {
    return planOf(&p->a).parts * p->a.q_rows * p->a.heads * (p->a.dim * static_cast<int64_t>(sizeof(float)) + static_cast<int64_t>(sizeof(float2)));
}

const char* mlkd_attention_kv4_kernel_names(const mlkd_attention_kv4* p) {
    static thread_local std::string name;
    const std::string type = typeName(p->a.dtype);
    const Plan n = planFor(p);
    if (!n.tiles) {
        name = "attentionKv4Rows<" + type + ">";
        return name.c_str();
    }
    const int dt = dimOf(p->a.dim);
    name = "attentionKv4Tiles<" + type + ", " + std::to_string(dt) + ", " + std::to_string(n.rows) + ", " + std::to_string(n.waves) + ">";
    if (n.parts > 0) name += "+attentionJoin<" + type + ", " + std::to_string(p->a.dim <= 64 ? 16 : p->a.dim <= 128 ? 32 : 64) + ">";
    return name.c_str();
}

int mlkd_launch_attention_kv4(const mlkd_attention_kv4* p, void* stream) {
    const int64_t rows = p->a.q_rows * p->a.heads;
    if (rows == 0) return 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (const Plan n = planFor(p); n.tiles) {
        const int rc = p->a.dtype == MLKD_F32   ? launchPlan<float>(p, n, st)
                       : p->a.dtype == MLKD_F16 ? launchPlan<_Float16>(p, n, st)
                                                : launchPlan<__bf16>(p, n, st);
        if (rc >= 0) return rc;   // else a grid past the limit
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 3) / 4, int64_t{1} << 20)));
    auto* kernel = p->a.dtype == MLKD_F32 ? attentionKv4Rows<float> : p->a.dtype == MLKD_F16 ? attentionKv4Rows<_Float16> : attentionKv4Rows<__bf16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, argsOf(p));
    return hipGetLastError() == hipSuccess ? 0 : MLKD_RT_LAUNCH;
}

}  // extern "C"
