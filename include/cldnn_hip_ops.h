/*
 * cldnn_hip_ops.h -- operators for image networks with attention, beside the convolution path of cldnn_hip.h: group norm
 * with an activation, matrix product with bias, activation and residual, rotary positions with several axes, attention.
 * The reference has none of them; they follow the manner of this layer.
 *
 * An operator is an object: create checks a description of the shapes, chooses the kernels and allocates the scratch
 * memory, enqueue launches on the engine's stream (asynchronous, device pointers, allocates nothing, may be recorded
 * with cldnn_hip_engine_record_begin or captured).  Calls of one object share its scratch and may not overlap.  Those made
 * through the library never do, whichever threads make them: the kernels of a call, and those of a recording, follow each
 * other on the engine's stream.  A graph that the application captured itself has to run on that stream too, and not be
 * launched while another thread enqueues the object.  A recording holds the operators whose memory its kernels use until
 * it is released; an operator in a graph that the application captured has to outlive the graph.  Every entry point
 * returns a cldnn_hip_status; the message of the last failure is cldnn_hip_last_error().  Exported by
 * libcldnn_hip_ops.so, which needs libcldnn_hip.so.
 *
 * Floating types: sums, statistics and softmax are held in 32 bits whatever the type of the data; results are rounded
 * once, to nearest even, unless stated otherwise.  Pointers need the alignment of one element; strides count elements.
 * Unless stated otherwise an output may not overlap an input.
 */
#ifndef CLDNN_HIP_OPS_H
#define CLDNN_HIP_OPS_H

#include "cldnn_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* data types beside those of cldnn_hip.h; its own entry points do not take them */
enum { CLDNN_HIP_F16 = 4, CLDNN_HIP_BF16 = 5 };

/* activations beside CLDNN_HIP_ACT_NONE, RELU, RELU_SLOPE and CLAMP; these entry points only */
enum {
    CLDNN_HIP_ACT_SILU = 4,      /* v / (1 + exp(-v)) */
    CLDNN_HIP_ACT_GELU = 5,      /* v * P(a standard normal value <= v) */
    CLDNN_HIP_ACT_GELU_TANH = 6  /* v / 2 * (1 + tanh(sqrt(2 / pi) * (v + 0.044715 v^3))) */
};

typedef struct cldnn_hip_operator_s* cldnn_hip_operator;

typedef struct {
    int32_t launches;          /* kernels per enqueue */
    int32_t grid, block;       /* of the first of them */
    int32_t lds_bytes;         /* of a workgroup: the most among them */
    int64_t workspace_bytes;   /* device memory that the object holds */
    int64_t ops;               /* floating-point operations of one call */
    int64_t bytes;             /* each input read once, each output written once (attention: of full lengths) */
    char kernel_name[96];      /* of all of them; products: for operands that are 16-byte aligned, others may take another */
} cldnn_hip_operator_info;

cldnn_hip_status cldnn_hip_operator_retain(cldnn_hip_operator op);
/* waits for the engine's stream: the scratch memory may be in use */
cldnn_hip_status cldnn_hip_operator_release(cldnn_hip_operator op);
cldnn_hip_status cldnn_hip_operator_get_info(cldnn_hip_operator op, cldnn_hip_operator_info* info);
/* cldnn_hip_tensor_bytes for tensors that may be of the types above; 0 on failure */
size_t cldnn_hip_operator_tensor_bytes(const cldnn_hip_tensor* t);

/* ------------------------------------------------------------------ group norm
 * Features in `groups` equal runs; per image and group, over its features and the whole plane,
 *   y = act((x - mean) / sqrt(variance + epsilon) * scale[f] + shift[f]),   variance = mean((x - mean)^2).
 * Tensors are byxf (channels last) of F32, F16 or BF16, input and output of any two of them; padding in any axis is a
 * stride here: it is neither read nor written.  The output may be the input (same pointer, same description). */
typedef struct {
    cldnn_hip_tensor input, output;   /* same logical sizes */
    int32_t groups;
    float epsilon;                    /* >= 0 */
    int32_t activation;               /* CLDNN_HIP_ACT_* */
    float activation_m, activation_n; /* RELU_SLOPE: m; CLAMP: [m, n] */
} cldnn_hip_group_norm_desc;
cldnn_hip_status cldnn_hip_group_norm_create(cldnn_hip_engine e, const cldnn_hip_group_norm_desc* desc, cldnn_hip_operator* out);
/* scale, shift: [f] float, NULL = 1 / 0 */
cldnn_hip_status cldnn_hip_group_norm_enqueue(cldnn_hip_operator op, const void* input_dev, const float* scale_dev, const float* shift_dev,
                                              void* output_dev);

/* ------------------------------------------------------------------ matrix product
 *   out[i][j] = act2(act(sum_k a[i][k] * weights[j][k] + bias[j]) + residual[i][j])
 * a: m rows of k, weights: n rows of k (as a fully_connected layer has them), F16 or BF16; the sum in 32 bits, rounded
 * once at the end.  The residual may lie in the output (same pointer, stride and type). */
typedef struct {
    int32_t m, n, k;
    int32_t dtype;                    /* of a and weights: CLDNN_HIP_F16 or BF16 */
    int32_t out_dtype;                /* dtype or CLDNN_HIP_F32 */
    int32_t residual_dtype;           /* dtype, CLDNN_HIP_F32, or CLDNN_HIP_NO_TYPE: none */
    int32_t has_bias;
    int64_t a_stride, weights_stride, out_stride, residual_stride; /* elements from row to row; 0 = dense */
    int32_t activation;               /* CLDNN_HIP_ACT_*, of the product with its bias */
    float activation_m, activation_n;
    int32_t residual_activation;      /* CLDNN_HIP_ACT_*, of the sum with the residual; NONE without one */
    float residual_activation_m, residual_activation_n;
} cldnn_hip_matmul_desc;
cldnn_hip_status cldnn_hip_matmul_create(cldnn_hip_engine e, const cldnn_hip_matmul_desc* desc, cldnn_hip_operator* out);
/* bias: [n] float; bias and residual are ignored (may be NULL) where the description has none */
cldnn_hip_status cldnn_hip_matmul_enqueue(cldnn_hip_operator op, const void* a_dev, const void* weights_dev, const float* bias_dev,
                                          const void* residual_dev, void* output_dev);

/* ------------------------------------------------------------------ rotary positions
 * Each head's first 2 * (pairs of all axes) values are pairs that turn with the token's position along one axis:
 *   angle = position[token][axis] * base^-(exponent),  y0 = x0 cos - x1 sin,  y1 = x1 cos + x0 sin;
 * the values behind them are copied.  Axis 0 has the first pairs, and so on.  The exponent of pair i, the j-th of its
 * axis' J, is j / J, or i / (pairs of all axes) with shared_frequencies.  Angles are good to 2^-24 of a turn for
 * positions up to 2^24 in magnitude; with a base below 1, whose frequencies go up to 1 / base, up to 2^24 * base. */
#define CLDNN_HIP_ROTARY_MAX_AXES 4
enum {
    CLDNN_HIP_ROTARY_INTERLEAVED = 0,     /* pair i: values 2i, 2i + 1 */
    CLDNN_HIP_ROTARY_HALVES = 1,          /* pair i: values i, i + (pairs of all axes) */
    CLDNN_HIP_ROTARY_HALVES_PER_AXIS = 2  /* the halves of the axis' own run of values */
};
typedef struct {
    int64_t tokens;                   /* of all images */
    int32_t q_heads, k_heads;         /* k_heads == 0: queries only */
    int32_t head_size;
    int32_t axes;
    int32_t pairs[CLDNN_HIP_ROTARY_MAX_AXES]; /* per axis; zero allowed */
    int32_t pairing;                  /* CLDNN_HIP_ROTARY_* */
    int32_t shared_frequencies;
    float base;
    int32_t dtype;                    /* CLDNN_HIP_F32, F16 or BF16 */
    int32_t position_dtype;           /* CLDNN_HIP_I32 or F32 */
    int32_t inverse;                  /* 1: turns back (the gradient of the forward form) */
    /* elements from token to token and from head to head; 0 = dense [tokens][heads][head_size] */
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
    int64_t q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride;
} cldnn_hip_rotary_desc;
cldnn_hip_status cldnn_hip_rotary_create(cldnn_hip_engine e, const cldnn_hip_rotary_desc* desc, cldnn_hip_operator* out);
/* positions: [tokens][axes].  An output may be its input (same pointer, same strides). */
cldnn_hip_status cldnn_hip_rotary_enqueue(cldnn_hip_operator op, const void* q_dev, const void* k_dev, const void* positions_dev,
                                          void* q_out_dev, void* k_out_dev);

/* ------------------------------------------------------------------ attention
 *   out[b][i][h] = sum_j softmax_j(scale * q[b][i][h] . k[b][j][g] + bias[b][h][i][j]) v[b][j][g],   g = h / (q_heads / kv_heads)
 * over the keys j < key_lengths[b] (clipped to 0..kv_len; all kv_len without lengths).  Keys and values at and behind a
 * length are never used, whatever their memory holds.  A row without a key, or with -infinity in all its scores, is
 * zeros.  The bias is ordinary arithmetic: -infinity takes a finite key out.  F16 or BF16; the softmax in 32 bits; the
 * probabilities are rounded to the data's type for the second product (and in BF16 their sum is that of the rounded ones).
 * head_size: a multiple of 8 up to 256; rows of q, k, v and out must be 16-byte aligned (pointers and strides). */
typedef struct {
    int32_t batch, q_len, kv_len, q_heads, kv_heads, head_size;  /* q_heads a multiple of kv_heads */
    int32_t dtype;
    float scale;                      /* 0 = 1 / sqrt(head_size); log2(e) times it has to be finite */
    int32_t has_key_lengths;
    int32_t bias_dtype;               /* dtype, CLDNN_HIP_F32, or CLDNN_HIP_NO_TYPE: none */
    /* elements; 0 = dense [batch][len][heads][head_size] */
    int64_t q_batch_stride, q_token_stride, q_head_stride;
    int64_t k_batch_stride, k_token_stride, k_head_stride;
    int64_t v_batch_stride, v_token_stride, v_head_stride;
    int64_t out_batch_stride, out_token_stride, out_head_stride;
    /* the bias is [..][kv_len] with these strides as they are: 0 = the same for every batch / head / query */
    int64_t bias_batch_stride, bias_head_stride, bias_q_stride;
} cldnn_hip_attention_desc;
cldnn_hip_status cldnn_hip_attention_create(cldnn_hip_engine e, const cldnn_hip_attention_desc* desc, cldnn_hip_operator* out);
/* key_lengths: [batch] int32; key_lengths and bias are ignored (may be NULL) where the description has none */
cldnn_hip_status cldnn_hip_attention_enqueue(cldnn_hip_operator op, const void* q_dev, const void* k_dev, const void* v_dev,
                                             const int32_t* key_lengths_dev, const void* bias_dev, void* output_dev);

#ifdef __cplusplus
}
#endif
#endif
