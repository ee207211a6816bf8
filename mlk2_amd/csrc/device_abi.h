// Plain-C launch descriptors shared by the C++ host planner and the HIP
// kernels. The host proves every address of a launch in bounds before it
// fills one of these; the device code never sees the Kernel IR itself.
#pragma once

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/// Element types a device buffer may hold (KernelBuffer::dtype subset,
/// compiler/include/mlk/type/domain.h:53-60).
/// BF16, I32, I8 and U8 are the operators' (mlkd_norm_rope and the ones below it).
enum mlkd_dtype { MLKD_F32 = 0, MLKD_F16 = 1, MLKD_F64 = 2, MLKD_BF16 = 3, MLKD_I32 = 4, MLKD_I8 = 5, MLKD_U8 = 6 };

/// Runtime scalar parameters of a chain (ScalarParam operands,
/// kernel_ir.h:58-70); indices past the bound table read 0.0 like the
/// reference evaluator (kernel_buffers.cpp:114-117).
enum { MLKD_MAX_SCALARS = 8 };
typedef struct mlkd_scalars {
    double v[MLKD_MAX_SCALARS];
} mlkd_scalars;

/// Row softmax / row sum: Y[r, :] = f(X[r, :]) over rows x cols, row strides
/// in elements.
typedef struct mlkd_softmax {
    const void* x;
    void* y;
    int32_t x_dtype, y_dtype;
    int64_t rows, cols;
    int64_t x_row_stride, y_row_stride;
    int32_t variant;     /* launch form; -1: the process default */
    int32_t pad;
} mlkd_softmax;

/// C[M,N] (+)= A[M,K] * B[K,N], row-major, leading dims in elements.
typedef struct mlkd_gemm {
    const void* a;
    const void* b;
    void* c;
    int32_t a_dtype, b_dtype, c_dtype;
    int32_t accumulate;   /* 1: C += A*B (Call form); 0: C = A*B */
    int64_t m, n, k;
    int64_t lda, ldb, ldc;
    int32_t variant;      /* launch form; -1: the process default */
    /* 1: skip the products of A[i,p] == 0, the reference's gemmRowBlock
       (kernel_buffers.cpp:422), with C[i,j] = C_in + sum over p ascending.
       With `accumulate`, the MFMA forms run it: a wave whose accumulators
       met an infinity or a NaN (only there can the skip change C) recomputes
       its block exactly. Otherwise the general kernel runs everything. */
    int32_t skip_zero_a;
    int32_t pad_;
    /* Device workspace for shapes the MFMA forms do not tile in whole blocks
       (mlkd_gemm_pad_bytes): operands whose rows are off 16 bytes are copied
       to aligned ones there, or the general kernel's K ranges leave their
       sums there. NULL (or too small) runs such shapes on the general kernel
       in one range. */
    void* work;
    int64_t work_bytes;
} mlkd_gemm;

/// S[b*seq + i, j] = softmax_j((Q[b,i,:] . K[b,j,:]) / div + bias[j]).
typedef struct mlkd_score_softmax {
    const void* q;
    const void* k;
    const void* bias;
    void* s;
    int32_t qk_dtype, bias_dtype, s_dtype;
    int32_t variant;      /* launch form; -1: the process default */
    int64_t batch, seq, dim;
    double div;
    /* Device scratch for the two-pass form's per-tile row statistics
       (mlkd_score_scratch_bytes); may be NULL, which selects another form. */
    void* scratch;
    int64_t scratch_bytes;
    /* Workspace for the row statistics of shapes that are not given scratch,
       or of more key ranges than it holds (mlkd_score_pad_bytes). NULL (or too
       small) keeps such shapes on the other kernels. */
    void* work;
    int64_t work_bytes;
} mlkd_score_softmax;

/// Head norms and position rotation of q and k, and k's and v's rows of a
/// cache. Row t of q, k, v: heads (kv_heads) heads of dim elements; strides
/// are elements from row to row. y = x / sqrt(mean x^2 + eps) * weight (no
/// weight: y = x), then the pairs of the first `rot` elements turned by
/// positions[axis, t] * theta^(-2 i / rot). Tokens t < tokens and, with
/// q_offsets, below q_offsets[sequences].
typedef struct mlkd_norm_rope {
    const void *q, *k, *v;               /* v may be NULL */
    void *q_out, *k_out, *v_out;
    const void *q_weight, *k_weight;     /* both or none */
    const int32_t* positions;            /* [axes, tokens], or NULL: no rotation */
    const int32_t* slots;                /* row of k_out and v_out, or NULL: row t */
    const int32_t* q_offsets;            /* [sequences + 1], or NULL */
    int32_t dtype, weight_dtype;
    int32_t heads, kv_heads, dim, rot;
    int32_t interleaved, axes, sequences, pad;
    int32_t section_end[3], pad2;        /* frequency pairs below which axis 0, 1, 2 applies */
    int64_t tokens, out_rows;            /* rows of q, k, v; rows of k_out and v_out */
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride, v_out_stride;
    double eps;
    double power[7];                     /* theta^(-2 2^k / rot): pair i turns by the product of its bits' powers */
} mlkd_norm_rope;

/// out = softmax(scale q k^T) v over packed sequences, and lse, the log of
/// each row's sum. Sequence b has query rows q_offsets[b] .. q_offsets[b + 1]
/// and keys kv_start[b] .. kv_start[b] + kv_len[b] (no arrays: its query rows);
/// with `prefix_k` every sequence's keys follow prefix rows 0 .. prefix_len.
/// Causal: query i of n sees own keys j <= i + kv_len - n. Lengths are clipped
/// to the buffers.
typedef struct mlkd_attention {
    const void *q, *k, *v, *prefix_k, *prefix_v;
    void* out;
    float* lse;                          /* [q_rows, heads], or NULL */
    const int32_t *q_offsets, *kv_start, *kv_len;
    const int32_t* prefix_len;           /* [1], or NULL: prefix_rows */
    int32_t dtype, causal;
    int32_t heads, kv_heads, dim, sequences;
    int64_t q_rows, kv_rows, prefix_rows;
    int64_t q_stride, k_stride, v_stride, prefix_k_stride, prefix_v_stride, out_stride;
    double scale;
    void* work;                          /* mlkd_attention_work_bytes, or NULL: no key ranges */
    int64_t work_bytes;
} mlkd_attention;

/// Rows in 8-bit integers: scale[t] = max |x[t, :]| / 127, codes[t, :] =
/// x[t, :] / scale[t] rounded to the nearest, half way to the even one, kept
/// within -127 .. 127. A row of zeros has scale 0 and codes 0, one that holds a
/// value that is not finite scale NaN and codes 0.
typedef struct mlkd_quantize_rows {
    const void* x;
    int8_t* codes;
    float* scale;                        /* [rows] */
    int32_t dtype, pad;                  /* of x */
    int64_t rows, cols;
    int64_t x_stride, codes_stride;      /* elements from row to row */
} mlkd_quantize_rows;

/// out[t, n] = (sum_k a[t, k] b[n, k]) a_scale[t] b_scale[n] + bias[n]; the sum
/// is exact (k < 2^17).
typedef struct mlkd_matmul_i8 {
    const int8_t *a, *b;
    const float *a_scale, *b_scale;      /* [m], [n] */
    const float* bias;                   /* [n], or NULL */
    void* out;
    int32_t dtype, pad;                  /* of out */
    int64_t m, n, k;
    int64_t lda, ldb, ldo;               /* elements from row to row */
    void* work;                          /* mlkd_matmul_i8_work_bytes, or NULL: no ranges of k */
    int64_t work_bytes;
} mlkd_matmul_i8;

/// Heads of k and v to and from the rows of a cache in 4 bits: a scale for each
/// row and head, max |x| / 6, and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to
/// |x| / scale, half way between two the one of the even code. A code is that
/// number's place, 0 .. 7, and 8 more where x has its sign bit set; element 2i
/// has the low half of byte i. A head of zeros has scale 0, one that holds a
/// value that is not finite scale NaN and codes 0. Token t takes row slots[t]
/// (row t without slots; rows outside the cache are left out), tokens below
/// q_offsets[sequences] only.
typedef struct mlkd_kv4_rows {
    void *k, *v;                         /* read by the store, written by the load */
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;            /* [cache_rows, kv_heads] */
    const int32_t* slots;                /* [tokens], or NULL */
    const int32_t* q_offsets;            /* [sequences + 1], or NULL */
    int32_t dtype, kv_heads, dim, sequences;
    int64_t tokens, cache_rows;
    int64_t k_stride, v_stride;          /* elements from row to row */
    int64_t k_codes_stride, v_codes_stride;   /* bytes from row to row */
} mlkd_kv4_rows;

/// mlkd_attention over such a cache: `a` with k and v the codes (strides in
/// bytes) and no prefix.
typedef struct mlkd_attention_kv4 {
    mlkd_attention a;
    const float *k_scale, *v_scale;      /* [kv_rows, kv_heads] */
} mlkd_attention_kv4;

#ifdef __cplusplus
}
#endif
