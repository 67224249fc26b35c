// C entry points of the int8 operators.
#include "ops_object.h"
#include "ops_s8.h"

using namespace chip;

extern "C" {

cldnn_hip_status cldnn_hip_quantize_create(cldnn_hip_engine e, const cldnn_hip_quantize_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_QUANTIZE, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.plan = quantize_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_quantize_enqueue(cldnn_hip_operator op, const void* input_dev, const float* factors_dev, void* output_dev, float* scales_dev)
{
    return guarded([&] {
        check_operator(op, OP_QUANTIZE);
        CHIP_REQUIRE(input_dev && output_dev && scales_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) { quantize_launch(s, *op->plan, input_dev, factors_dev, output_dev, scales_dev); });
    });
}

cldnn_hip_status cldnn_hip_matmul_s8_create(cldnn_hip_engine e, const cldnn_hip_matmul_s8_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_MATMUL_S8, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.plan = matmul_s8_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_matmul_s8_enqueue(cldnn_hip_operator op, const void* a_dev, const void* weights_dev, const float* a_scales_dev,
                                             const float* weights_scales_dev, const float* bias_dev, const void* residual_dev, void* output_dev)
{
    return guarded([&] {
        check_operator(op, OP_MATMUL_S8);
        CHIP_REQUIRE(a_dev && weights_dev && output_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) {
            matmul_s8_launch(s, *op->plan, op->workspace, a_dev, weights_dev, a_scales_dev, weights_scales_dev, bias_dev, residual_dev, output_dev);
        });
    });
}

cldnn_hip_status cldnn_hip_block_norm_create(cldnn_hip_engine e, const cldnn_hip_block_norm_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_BLOCK_NORM, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.plan = block_norm_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_block_norm_enqueue(cldnn_hip_operator op, const void* x_dev, const void* branch_dev, const float* post_weight_dev,
                                              const float* post_bias_dev, const void* gate_dev, const float* weight_dev, const float* bias_dev,
                                              const void* scale_dev, const void* shift_dev, void* y_dev, void* output_dev, float* out_scales_dev)
{
    return guarded([&] {
        check_operator(op, OP_BLOCK_NORM);
        CHIP_REQUIRE(x_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) {
            block_norm_launch(s, *op->plan, {x_dev, branch_dev, post_weight_dev, post_bias_dev, gate_dev, weight_dev, bias_dev, scale_dev, shift_dev, y_dev, output_dev, out_scales_dev});
        });
    });
}

}  // extern "C"
