/*
 * cldnn_hip_ops_s8.h -- operators that bring the transformer blocks of an image network into int8, beside the float operators of
 * cldnn_hip_ops.h: rows quantised with a scale each, the matrix product of int8 operands with scales for each token and channel,
 * and the norms before and after a block with its gate and residual scale, whose result may be int8 too.
 *
 * The reference has none of them.  Objects, scratch memory, streams, recordings, threads, errors, alignment and overlap are as in
 * cldnn_hip_ops.h, and cldnn_hip_operator_retain, _release and _get_info serve these objects as well.  Exported by
 * libcldnn_hip_ops_s8.so, which needs libcldnn_hip_ops.so and libcldnn_hip.so.
 *
 * A quantised row: 8-bit whole numbers q and one float, scale; the values it stands for are q * scale.  Of values y it is
 *   most = max |y|,   scale = most / 127,   q = y * (127 / most) rounded to the nearest whole number, ties to even,
 * each quotient and product rounded to 32 bits; |q| <= 127.  A row whose `most` is below 2^-120 counts as zeros (scale 0).  A row with
 * a NaN or an infinity gets q = 0 and scale NaN, so that every product of the row is NaN.
 *
 * CLDNN_HIP_ACT_GELU is worked out to within 1.5e-7 |v|, which far below zero may be as much as the value: a row of nothing but such v
 * becomes the quantised row of what was worked out.
 */
#ifndef CLDNN_HIP_OPS_S8_H
#define CLDNN_HIP_OPS_S8_H

#include "cldnn_hip_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ rows to int8
 * A row of x becomes a quantised row of
 *   y[f] = act(x[f]) * factor[f],   gated:  y[f] = act(x[f]) * x[features + f] * factor[f]   (the input has 2 * features values)
 * Serves activations (a row is a token) as well as weights (a row is an output channel). */
typedef struct {
    int64_t rows;
    int32_t features;                 /* of the output */
    int32_t dtype;                    /* of the input: CLDNN_HIP_F32, F16 or BF16 */
    int32_t gated;
    int32_t has_factors;
    int32_t activation;               /* CLDNN_HIP_ACT_* */
    float activation_m, activation_n;
    int64_t in_stride, out_stride;    /* elements from row to row; 0 = dense */
} cldnn_hip_quantize_desc;
cldnn_hip_status cldnn_hip_quantize_create(cldnn_hip_engine e, const cldnn_hip_quantize_desc* desc, cldnn_hip_operator* out);
/* factors: [features] float, ignored (may be NULL) where the description has none; output: int8; scales: [rows] float */
cldnn_hip_status cldnn_hip_quantize_enqueue(cldnn_hip_operator op, const void* input_dev, const float* factors_dev, void* output_dev, float* scales_dev);

/* ------------------------------------------------------------------ matrix product of int8 operands
 *   out[i][j] = act2(act(sum_k a[i][k] * weights[j][k] * a_scale[i] * weights_scale[j] + bias[j]) + residual[i][j])
 * a: m rows of k int8, weights: n rows of k int8.  The sum is exact; it is rounded to 32 bits, multiplied by the row's scale, then by the
 * channel's, and the result rounded once at the end.  The residual may lie in the output (same pointer, stride and type).
 * Operands that are not aligned to 16 bytes take smaller tiles: enqueue refuses them (CLDNN_HIP_UNSUPPORTED_SIZE) where the result has
 * 2^24 tiles of 64 x 64 or more. */
enum {
    CLDNN_HIP_SCALES_NONE = 0,        /* 1 */
    CLDNN_HIP_SCALES_ONE = 1,         /* one for all rows */
    CLDNN_HIP_SCALES_EACH = 2         /* one to a row */
};
typedef struct {
    int32_t m, n, k;                  /* k at most 131071: sums of that many products fit 32 bits */
    int32_t a_scales, weights_scales; /* CLDNN_HIP_SCALES_*, of the rows of a and of the weights */
    int32_t out_dtype;                /* CLDNN_HIP_F32, F16 or BF16 */
    int32_t residual_dtype;           /* the same, or CLDNN_HIP_NO_TYPE: none */
    int32_t has_bias;
    int64_t a_stride, weights_stride, out_stride, residual_stride; /* elements from row to row; 0 = dense */
    int32_t activation;               /* CLDNN_HIP_ACT_*, of the product with its bias */
    float activation_m, activation_n;
    int32_t residual_activation;      /* CLDNN_HIP_ACT_*, of the sum with the residual; NONE without one */
    float residual_activation_m, residual_activation_n;
} cldnn_hip_matmul_s8_desc;
cldnn_hip_status cldnn_hip_matmul_s8_create(cldnn_hip_engine e, const cldnn_hip_matmul_s8_desc* desc, cldnn_hip_operator* out);
/* a_scales, weights_scales: float, one or one to a row; bias: [n] float; each is ignored (may be NULL) where the description has none */
cldnn_hip_status cldnn_hip_matmul_s8_enqueue(cldnn_hip_operator op, const void* a_dev, const void* weights_dev, const float* a_scales_dev,
                                             const float* weights_scales_dev, const float* bias_dev, const void* residual_dev, void* output_dev);

/* ------------------------------------------------------------------ norms before and after a block
 * Between two blocks of a residual network, for each token (x: the stream, branch: what the block before gave):
 *   z = post(branch) * post_weight + post_bias
 *   y = residual_scale * x + gate * z                                  the stream behind the block
 *   h = (norm(y) * weight + bias) * (1 + scale) + shift                what the next block reads
 * post, norm: (v - mean) / sqrt(variance + epsilon), v / sqrt(mean of v^2 + epsilon), or v.  Weights and biases are [features] float, the
 * same for all tokens; gate, scale and shift are [images][features], one row for tokens_per_image tokens one behind the other.  h is made
 * of y in 32 bits, before y is rounded to the stream's type.  Statistics are of values that a thread group holds: the mean first, then the
 * squares around it. */
enum {
    CLDNN_HIP_TOKEN_NORM_NONE = 0,
    CLDNN_HIP_TOKEN_NORM_LAYER = 1,
    CLDNN_HIP_TOKEN_NORM_RMS = 2
};
typedef struct {
    int64_t tokens;                   /* of all images */
    int32_t features;                 /* at most 32768 */
    int32_t tokens_per_image;         /* 0: all tokens share one row of gate, scale and shift */
    int32_t dtype;                    /* of the stream, x and y: CLDNN_HIP_F32, F16 or BF16 */
    int32_t branch_dtype;             /* the same, or CLDNN_HIP_NO_TYPE: no branch; y is x then, and not written */
    int32_t out_dtype;                /* of h: F32, F16, BF16, CLDNN_HIP_S8 (quantised rows), or CLDNN_HIP_NO_TYPE: only y is wanted */
    int32_t modulation_dtype;         /* of gate, scale and shift: F32, F16, BF16, or CLDNN_HIP_NO_TYPE: none */
    int32_t norm, post;               /* CLDNN_HIP_TOKEN_NORM_*; post: NONE without a branch, norm: NONE where only y is wanted */
    float epsilon, post_epsilon;      /* >= 0 */
    float residual_scale;             /* 1 without a branch */
    /* elements from token to token, of gate, scale and shift from image to image; 0 = dense */
    int64_t x_stride, branch_stride, y_stride, out_stride, gate_stride, scale_stride, shift_stride;
} cldnn_hip_block_norm_desc;
cldnn_hip_status cldnn_hip_block_norm_create(cldnn_hip_engine e, const cldnn_hip_block_norm_desc* desc, cldnn_hip_operator* out);
/* post_weight, weight, gate: NULL = 1; post_bias, bias, scale, shift: NULL = 0.  y: NULL = not wanted, may be x (same pointer, same
 * stride).  out_scales: [tokens] float, of quantised rows.  What the description has not is ignored (may be NULL). */
cldnn_hip_status cldnn_hip_block_norm_enqueue(cldnn_hip_operator op, const void* x_dev, const void* branch_dev, const float* post_weight_dev,
                                              const float* post_bias_dev, const void* gate_dev, const float* weight_dev, const float* bias_dev,
                                              const void* scale_dev, const void* shift_dev, void* y_dev, void* output_dev, float* out_scales_dev);

#ifdef __cplusplus
}
#endif
#endif
