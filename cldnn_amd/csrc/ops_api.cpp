// C entry points of the float operators: objects, their scratch memory, checks of pointers.
#include <cstring>
#include <memory>
#include <vector>

#include "ops_object.h"

using namespace chip;

cldnn_hip_operator_s::~cldnn_hip_operator_s()
{
    free_plan(norm);
    free_plan(matmul);
    free_plan(rotary);
    free_plan(attention);
}

extern "C" {

cldnn_hip_status cldnn_hip_operator_retain(cldnn_hip_operator op)
{
    return guarded([&] {
        CHIP_REQUIRE(op, CLDNN_HIP_INVALID_ARG, "null operator");
        op->refs.fetch_add(1);
    });
}

cldnn_hip_status cldnn_hip_operator_release(cldnn_hip_operator op)
{
    return guarded([&] {
        CHIP_REQUIRE(op, CLDNN_HIP_INVALID_ARG, "null operator");
        if (op->refs.fetch_sub(1) != 1) return;
        if (op->workspace) {
            (void)hipSetDevice(op->engine->device);
            (void)hipStreamSynchronize(op->engine->stream);
        }
        DiscardOperator()(op);
    });
}

cldnn_hip_status cldnn_hip_operator_get_info(cldnn_hip_operator op, cldnn_hip_operator_info* info)
{
    return guarded([&] {
        CHIP_REQUIRE(op && info, CLDNN_HIP_INVALID_ARG, "null argument");
        *info = op->info;
    });
}

size_t cldnn_hip_operator_tensor_bytes(const cldnn_hip_tensor* t)
{
    size_t bytes = 0;
    (void)guarded([&] {
        CHIP_REQUIRE(t, CLDNN_HIP_INVALID_ARG, "null tensor");
        const bool half = t->dtype == CLDNN_HIP_F16 || t->dtype == CLDNN_HIP_BF16;
        bytes = tensor_elems(*t) * (half ? 2 : dtype_size(t->dtype));
    });
    return bytes;
}

cldnn_hip_status cldnn_hip_group_norm_create(cldnn_hip_engine e, const cldnn_hip_group_norm_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_GROUP_NORM, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.norm = norm_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_group_norm_enqueue(cldnn_hip_operator op, const void* input_dev, const float* scale_dev, const float* shift_dev,
                                              void* output_dev)
{
    return guarded([&] {
        check_operator(op, OP_GROUP_NORM);
        CHIP_REQUIRE(input_dev && output_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) { norm_launch(s, *op->norm, op->workspace, input_dev, scale_dev, shift_dev, output_dev); });
    });
}

cldnn_hip_status cldnn_hip_matmul_create(cldnn_hip_engine e, const cldnn_hip_matmul_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_MATMUL, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.matmul = matmul_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_matmul_enqueue(cldnn_hip_operator op, const void* a_dev, const void* weights_dev, const float* bias_dev,
                                          const void* residual_dev, void* output_dev)
{
    return guarded([&] {
        check_operator(op, OP_MATMUL);
        CHIP_REQUIRE(a_dev && weights_dev && output_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) { matmul_launch(s, *op->matmul, op->workspace, a_dev, weights_dev, bias_dev, residual_dev, output_dev); });
    });
}

cldnn_hip_status cldnn_hip_rotary_create(cldnn_hip_engine e, const cldnn_hip_rotary_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_ROTARY, [&](cldnn_hip_operator_s& op, std::vector<char>& init) { op.rotary = rotary_plan(*e, *desc, op.info, init); });
}

cldnn_hip_status cldnn_hip_rotary_enqueue(cldnn_hip_operator op, const void* q_dev, const void* k_dev, const void* positions_dev,
                                          void* q_out_dev, void* k_out_dev)
{
    return guarded([&] {
        check_operator(op, OP_ROTARY);
        CHIP_REQUIRE(q_dev && q_out_dev && positions_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) { rotary_launch(s, *op->rotary, op->workspace, q_dev, k_dev, positions_dev, q_out_dev, k_out_dev); });
    });
}

cldnn_hip_status cldnn_hip_attention_create(cldnn_hip_engine e, const cldnn_hip_attention_desc* desc, cldnn_hip_operator* out)
{
    return create_operator(e, desc, out, OP_ATTENTION, [&](cldnn_hip_operator_s& op, std::vector<char>&) { op.attention = attention_plan(*e, *desc, op.info); });
}

cldnn_hip_status cldnn_hip_attention_enqueue(cldnn_hip_operator op, const void* q_dev, const void* k_dev, const void* v_dev,
                                             const int32_t* key_lengths_dev, const void* bias_dev, void* output_dev)
{
    return guarded([&] {
        check_operator(op, OP_ATTENTION);
        CHIP_REQUIRE(q_dev && k_dev && v_dev && output_dev, CLDNN_HIP_INVALID_ARG, "null device pointer");
        enqueue_operator(op, [&](hipStream_t s) { attention_launch(s, *op->attention, op->workspace, q_dev, k_dev, v_dev, key_lengths_dev, bias_dev, output_dev); });
    });
}

}  // extern "C"
