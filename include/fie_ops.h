/*
 * fie_ops.h -- C ABI of the operators in front of the output layer and of the output layer
 * in 8-bit integers: block norms, per-token quantisation, the integer product.  No
 * counterpart on the reference's sampler path.
 *
 * Conventions are fie_sampler.h's: device pointers, work enqueued on `stream`, nothing
 * synchronises or allocates, FIE_OK or a negative FIE_E* code, and
 * fie_sampler_last_error() holds the message.
 */
#ifndef FIE_OPS_H
#define FIE_OPS_H

#include "fie_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { FIE_I8 = 3 };            /* beside FIE_F32, FIE_F16, FIE_BF16 */

enum { FIE_NORM_RMS = 0, FIE_NORM_LAYER = 1, FIE_NORM_NONE = 2 };

/* One row a token, `width` wide, all in fp32 between the loads and the stores:
     z = x                                          (no x: no z)
     z = norm(z) * (post_weight + weight_offset) + post_bias     (with post_norm)
     z = z * gate                                   (with a gate)
     r = residual + scale * z
     y = norm(r) * (weight + weight_offset) + bias  (kind FIE_NORM_NONE: y = r)
   norm is v / sqrt(mean(v^2) + eps), or with FIE_NORM_LAYER the same of v - mean(v).
   Absent weights are 1 (without the offset), absent biases 0.  r is rounded into
   residual_out, y is taken from the unrounded r.  With y_dtype FIE_I8, y is stored as
   round(y / s), at most 127 either way, s = max|y| / 127 of its row in y_scale (an all-zero
   row: 0 and s = 0; a row with a NaN: 0 and s = NaN, one with an infinity: 0 and s infinite, so that
   the product's row is NaN in both). */
typedef struct fie_norm_args {
    const void* x;              /* [tokens, width], or NULL */
    const void* residual;       /* [tokens, width] */
    void* residual_out;         /* [tokens, width] in residual_dtype, or NULL; may be `residual` */
    void* y;                    /* [tokens, width], or NULL */
    float* y_scale;             /* [tokens], with FIE_I8 */
    const void* weight;         /* [width] in x_dtype, or fp32 with weight_f32; likewise: */
    const void* bias;
    const void* post_weight;
    const void* post_bias;
    const void* gate;           /* [tokens or 1, width or 1] in x_dtype, or fp32 with gate_f32 */
    int64_t tokens;
    int64_t x_stride, residual_stride, residual_out_stride, y_stride;   /* elements between rows */
    int64_t gate_stride;        /* 0: one row for every token */
    int32_t gate_step;          /* 1, or 0: one value for a whole row */
    int32_t width;              /* 1..FIE_MAX_WIDTH (FIE_MAX_K: kind NONE of a residual alone to FIE_I8) */
    int32_t x_dtype;            /* of x and y (without x: of y's float type); FIE_F32, F16, BF16 */
    int32_t residual_dtype;     /* x_dtype or FIE_F32 (without x: any of the three) */
    int32_t y_dtype;            /* x_dtype or FIE_I8 */
    int32_t weight_f32, gate_f32;
    int32_t kind;               /* FIE_NORM_* */
    int32_t post_norm;          /* 1: z is normed (kind's norm, not FIE_NORM_NONE) */
    float scale, eps, weight_offset;
} fie_norm_args;
#define FIE_MAX_WIDTH 65536

int fie_block_norm(const fie_norm_args* args, void* stream);

/* y[m, n] = x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] + bias[n]: int32 sums (exact),
   fp32 scaling, one rounding to y_dtype. */
typedef struct fie_int8_args {
    const int8_t* x;            /* [m, k], rows x_stride bytes apart */
    const int8_t* w;            /* [n, k], rows w_stride bytes apart (nn.Linear's layout) */
    const float* x_scale;       /* [m] */
    const float* w_scale;       /* [n] */
    const float* bias;          /* [n] or NULL */
    void* y;                    /* [m, n], rows y_stride elements apart */
    int64_t m, x_stride, w_stride, y_stride;
    int32_t n, k;               /* 1 <= k <= FIE_MAX_K (the sums stay in 32 bits) */
    int32_t y_dtype;            /* FIE_F32, FIE_F16, FIE_BF16 */
    int32_t reserved;
    void* workspace;            /* fie_int8_workspace_size() bytes, 16-byte aligned (NULL: none) */
    size_t workspace_bytes;
} fie_int8_args;
#define FIE_MAX_K 131071

/* Bytes that a call with these pointers and sizes needs beside its operands: 0 where the rows
   of x and w begin at multiples of 16 bytes (and for few tokens); otherwise the unaligned
   operand is laid out there first.  Weights whose rows are padded to 16 bytes avoid that. */
size_t fie_int8_workspace_size(const fie_int8_args* args);

int fie_int8_linear(const fie_int8_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FIE_OPS_H */
