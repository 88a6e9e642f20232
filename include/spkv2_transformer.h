/*
 * Operators of an INT8 decoder layer on device tensors (B200, sm_100a).
 *
 * They have no counterpart in the reference runtime, whose packages hold
 * static graphs: a decoder's batch, lengths and encoder states change from
 * call to call, so these are plain calls on device pointers, next to the
 * graph runtime whose image features they read.
 *
 *   spkv2_cuda_rms_norm_i8        residual addition, root-mean-square norm,
 *                                 int8 codes and a scale for each token
 *   spkv2_cuda_quantize_rows_i8   int8 codes and a scale for each row
 *   spkv2_cuda_dequantize_rows_i8 the values that codes stand for
 *   spkv2_cuda_linear_i8          int8 x int8 product with a scale for each
 *                                 token and each channel, bias, activation
 *   spkv2_cuda_cross_attention    attention of queries to an encoder's keys
 *                                 and values of another length
 *
 * Conventions of all of them:
 *   - Every pointer is device memory of the current device.  Strides count
 *     elements; the last dimension is contiguous.  A pointer or stride that
 *     is not a multiple of 16 bytes is served, by a slower kernel; a pointer
 *     that is not a multiple of its element's size is a bad argument.
 *   - The call checks its arguments on the host, launches one kernel on
 *     `stream` (a cudaStream_t; NULL = legacy default stream) and returns.
 *     It allocates nothing, keeps nothing and can be captured into a graph.
 *   - It returns 0, -1 (bad argument), SPKV2_ERR_UNSUPPORTED (type or size
 *     outside the ranges below) or a CUDA-target error code
 *     (spkv2_cuda.h).  Calls with nothing to write return 0.
 *   - Sums, norms, softmax statistics and accumulators are fp32 or int32 (fp64
 *     for the scale of a row whose squares leave fp32's range); a result is
 *     rounded when it is stored.  Two roundings come before: cross_attention
 *     rounds each probability to a 16-bit type of its inputs, as both operands
 *     of a tensor-core product have one type, and adds them up unrounded; codes
 *     are y times a reciprocal, so a value that lies midway between two codes, to
 *     2^-14 of a step, may take either.
 *   - Results do not depend on timing: the same call gives the same bits.
 */
#ifndef SPKV2_TRANSFORMER_H
#define SPKV2_TRANSFORMER_H

#include <stdint.h>
#include "spkv2_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Element types: SPKV2_DTYPE_FP32 and SPKV2_DTYPE_FP16 of the package format,
 * and bfloat16, which packages do not hold. */
#define SPKV2_CUDA_DTYPE_BF16 16

/* linear_i8's activation: the codes of the fused activations of a Conv.  ReLU
 * keeps a NaN. */
#define SPKV2_CUDA_ACT_NONE 0
#define SPKV2_CUDA_ACT_RELU 1
#define SPKV2_CUDA_ACT_SILU 2

/* s = x + residual;  y = s * weight / sqrt(mean(s^2) + eps);
 * scale = max|y| / 127;  codes = round_half_even(y / scale), per row.
 * A row of zeros has scale 0 and codes 0; a row whose s (an fp32 sum) or
 * weight holds an infinity or a NaN has scale NaN and codes 0.  Finite rows may
 * lie anywhere in fp32's range, squares beyond it included; weights other than
 * 0 from 2^-64 to 2^64.  sum (if given) receives s in x's type and may be x or
 * residual itself.  width: 1 .. 2^24. */
typedef struct {
    const void *x;        /* [rows, width] */
    const void *residual; /* [rows, width] in x's type, or NULL */
    const void *weight;   /* [width] in x's type */
    void *sum;            /* [rows, width] in x's type, or NULL */
    int8_t *codes;        /* [rows, width] */
    float *scale;         /* [rows] */
    int64_t rows, width;
    int64_t x_stride, residual_stride, sum_stride, codes_stride; /* between rows */
    float eps;
    int32_t dtype; /* of x */
} Spkv2RmsNormI8;

int spkv2_cuda_rms_norm_i8(const Spkv2RmsNormI8 *args, void *stream);

/* scale = max|x| / 127;  codes = round_half_even(x / scale), per row, with the
 * rules above for rows of zeros and rows that are not finite.  Applied to a
 * weight [channels, width] it gives linear_i8's weight and channel scales. */
typedef struct {
    const void *x; /* [rows, width] */
    int8_t *codes;
    float *scale;
    int64_t rows, width;
    int64_t x_stride, codes_stride;
    int32_t dtype; /* of x */
    int32_t reserved;
} Spkv2QuantizeRowsI8;

int spkv2_cuda_quantize_rows_i8(const Spkv2QuantizeRowsI8 *args, void *stream);

/* y = codes * scale[row]. */
typedef struct {
    const int8_t *codes; /* [rows, width] */
    const float *scale;  /* [rows] */
    void *y;             /* [rows, width] */
    int64_t rows, width;
    int64_t codes_stride, y_stride;
    int32_t dtype; /* of y */
    int32_t reserved;
} Spkv2DequantizeRowsI8;

int spkv2_cuda_dequantize_rows_i8(const Spkv2DequantizeRowsI8 *args, void *stream);

/* y[i, j] = act(float(sum_k a[i, k] * w[j, k]) * a_scale[i] * w_scale[j] + bias[j]);
 * the sum is exact in int32 (k <= 131071). */
typedef struct {
    const int8_t *a;      /* [m, k] */
    const float *a_scale; /* [m] */
    const int8_t *w;      /* [n, k] */
    const float *w_scale; /* [n] */
    const float *bias;    /* [n], or NULL */
    void *y;              /* [m, n] */
    int64_t m, n, k;
    int64_t a_stride, w_stride, y_stride; /* between rows */
    int32_t dtype;                        /* of y */
    int32_t activation;
} Spkv2LinearI8;

int spkv2_cuda_linear_i8(const Spkv2LinearI8 *args, void *stream);

/* out[b, i, h] = sum_j p_j v[b, j, h / (heads / kv_heads)],
 * p = softmax over the keys j that count of scale * <q[b, i, h], k[b, j, ...]>.
 * Key j of entry b counts if j < lengths[b] (where lengths is given; values
 * outside 0 .. keys are clamped) and key_mask[b, j] != 0 (where it is given).
 * What lies in the keys and values that do not count has no influence, NaN
 * included.  A row without keys is 0.  heads is a multiple of kv_heads;
 * width: 1 .. 256, the same for keys and values.  A stride of 0 stands for one
 * place for all, in the inputs only. */
typedef struct {
    const void *q;           /* [batch, queries, heads, width] */
    const void *k;           /* [batch, keys, kv_heads, width] in q's type */
    const void *v;           /* [batch, keys, kv_heads, width] in q's type */
    void *out;               /* [batch, queries, heads, width] in q's type */
    const int32_t *lengths;  /* [batch], or NULL */
    const uint8_t *key_mask; /* [batch, keys], or NULL */
    int64_t batch, queries, keys;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3]; /* batch, token, head */
    int64_t mask_stride;                                          /* between entries */
    int32_t heads, kv_heads, width;
    int32_t dtype; /* of q */
    float scale;
    int32_t reserved;
} Spkv2CrossAttention;

int spkv2_cuda_cross_attention(const Spkv2CrossAttention *args, void *stream);

/* Every wait for data inside the kernels (on an mbarrier) has a limit of about a
 * second; the barriers of a cluster and the allocation of tensor memory wait for
 * CTAs of the GPU only, without one.  A wait that runs out records a role code (2 operand loads, 3 matrix products, 4 results, 7
 * hand-over) on the device and lets its kernel return, with its outputs
 * incomplete.  This call waits for the current device's work and returns 0, or
 * SPKV2_ERR_DEVICE_STATUS with the first such code since the last call. */
int spkv2_cuda_transformer_status(int *code);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* SPKV2_TRANSFORMER_H */
