// What the int8 operators' library shares: plans, launches.
#pragma once
#include "../../include/cldnn_hip_ops_s8.h"
#include "ops_common.h"

namespace chip {

// Each: what create works out from a description (refusing what is wrong), and the launch.
std::unique_ptr<OperatorPlan> quantize_plan(const cldnn_hip_engine_s& e, const cldnn_hip_quantize_desc& d, cldnn_hip_operator_info& info);
void quantize_launch(hipStream_t s, const OperatorPlan& p, const void* in, const float* factors, void* out, float* scales);
std::unique_ptr<OperatorPlan> matmul_s8_plan(const cldnn_hip_engine_s& e, const cldnn_hip_matmul_s8_desc& d, cldnn_hip_operator_info& info);
void matmul_s8_launch(hipStream_t s, const OperatorPlan& p, void* workspace, const void* a, const void* w, const float* a_scales, const float* w_scales, const float* bias,
                      const void* residual, void* out);
std::unique_ptr<OperatorPlan> block_norm_plan(const cldnn_hip_engine_s& e, const cldnn_hip_block_norm_desc& d, cldnn_hip_operator_info& info);
// what a call of a block norm is given
struct BlockNormPointers {
    const void *x, *branch;
    const float *post_weight, *post_bias;
    const void* gate;
    const float *weight, *bias;
    const void *scale, *shift;
    void *y, *out;
    float* out_scales;
};
void block_norm_launch(hipStream_t s, const OperatorPlan& p, const BlockNormPointers& of);

}  // namespace chip
