// Norms before and after a block, with its gate and residual scale:
//   z = post(branch) * post_weight + post_bias,  y = residual_scale * x + gate * z,  h = (norm(y) * weight + bias) * (1 + scale) + shift
//
// One pass: a token's row is read once and held in registers; the mean is taken first, then the squares around it, so that a mean far
// from zero costs no digits.  Bound by memory: 25088 x 1024 in bf16, a branch with gate, scale and shift, 206 MB, 44 us, 4.7 TB/s; 784 x
// 8192 of an f32 stream with an f16 branch, norms on both sides, 77 MB, 16.6 us, 4.6 TB/s.  Narrow rows, 16 threads to each, 12 of which have
// a vector: 100352 x 96 in bf16, as the first, 77 MB, 21 us, 3.7 TB/s; 100352 x 128, 103 MB, 22 us, 4.7.  One token takes a launch, 3 us.
#include "row_kernel.h"

namespace chip {

struct BlockNormArgs {
    int64_t tokens;
    int32_t C, per_image;  // per_image 0: one image
    int32_t x_type, branch_type, out_type, mod_type;
    int32_t norm, post;
    float epsilon, post_epsilon, residual_scale;
    int32_t past_y, past_out;  // results that go past the caches
    int64_t x_pitch, branch_pitch, y_pitch, out_pitch, gate_pitch, scale_pitch, shift_pitch;
};

namespace {
struct BlockNormPlan : OperatorPlan {
    BlockNormArgs a{};
    RowShape shape{};
};
}  // namespace

__device__ inline int block_norm_size(int type) { return type == CLDNN_HIP_S8 ? 1 : type == CLDNN_HIP_F32 ? 4 : 2; }

// The values of a row, zeros where they are not the lane's, become their unit form; two slots of LDS.
template <int LANES, int NV, int SURE>
__device__ __forceinline__ void block_norm_unit(float (&v)[NV][8], int kind, int C, float epsilon, int lane, float (*slot)[LANES < 64 ? 1 : LANES / 64])
{
    if (kind == CLDNN_HIP_TOKEN_NORM_NONE) return;
    const auto each = [&](auto&& f) __attribute__((always_inline)) { row_each<LANES, NV, SURE>(lane, C, f); };
    if (kind == CLDNN_HIP_TOKEN_NORM_LAYER) {
        float sum = 0.0f;
        each([&](int i, RowVector) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += v[i][j];
        });
        const float mean = row_sum<LANES>(sum, slot[0]) / (float)C;
        each([&](int i, RowVector of) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] -= mean;
            row_mask(of, C, v[i]);
        });
    }
    float squares = 0.0f;
    each([&](int i, RowVector) {
#pragma unroll
        for (int j = 0; j < 8; ++j) squares = __builtin_fmaf(v[i][j], v[i][j], squares);
    });
    const float factor = 1.0f / __builtin_sqrtf(row_sum<LANES>(squares, slot[1]) / (float)C + epsilon);
    each([&](int i, RowVector) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= factor;
    });
}

template <int LANES, int NV, int SURE>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES, row_waves(NV)) void block_norm_kernel(BlockNormArgs a, BlockNormPointers p)
{
    constexpr int THREADS = LANES < 256 ? 256 : LANES;
    __shared__ float slot[5][LANES < 64 ? 1 : LANES / 64];
    const int lane = threadIdx.x & (LANES - 1), C = row_length<LANES, SURE>(a.C);
    const int64_t row = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    if (row >= a.tokens) return;  // whole groups: nobody waits for them
    const int64_t image = a.per_image ? (uint32_t)row / (uint32_t)a.per_image : 0;
    const auto at = [](const void* base, int64_t elements, int type) { return (const char*)base + elements * block_norm_size(type); };
    const auto each = [&](auto&& f) __attribute__((always_inline)) { row_each<LANES, NV, SURE>(lane, C, f); };
    const bool has_branch = a.branch_type != CLDNN_HIP_NO_TYPE;
    RowRaw<true> x[NV], branch[NV];
    const char *x_row = at(p.x, row * a.x_pitch, a.x_type), *branch_row = at(p.branch, row * a.branch_pitch, a.branch_type);
    if (has_branch) each([&](int i, RowVector of) { branch[i] = row_load<true>(branch_row, a.branch_type, of.c, C); });
    each([&](int i, RowVector of) { x[i] = row_load<true>(x_row, a.x_type, of.c, C); });
    float v[NV][8];
    const auto times = [&](int i, const float (&f)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= f[j];
    };
    const auto plus = [&](int i, const float (&f)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += f[j];
    };
    // a vector of the image's row of gate, scale or shift
    const auto modulation = [&](const void* base, int64_t pitch, int c, float (&f)[8]) { row_values(row_load<true>(at(base, image * pitch, a.mod_type), a.mod_type, c, C), a.mod_type, f); };
    if (has_branch) {
        each([&](int i, RowVector of) { row_values(branch[i], a.branch_type, v[i]), row_mask(of, C, v[i]); });
        block_norm_unit<LANES, NV, SURE>(v, a.post, C, a.post_epsilon, lane, slot);
        each([&](int i, RowVector of) {
            float f[8];
            if (p.post_weight) row_floats(p.post_weight, of.c, C, f), times(i, f);
            if (p.post_bias) row_floats(p.post_bias, of.c, C, f), plus(i, f);
            if (p.gate) modulation(p.gate, a.gate_pitch, of.c, f), times(i, f);
            row_values(x[i], a.x_type, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = __builtin_fmaf(a.residual_scale, f[j], v[i][j]);
            if (p.y) {
                char* y_row = (char*)p.y + row * a.y_pitch * block_norm_size(a.x_type);
                if (a.past_y) row_store<true>(y_row, a.x_type, of, C, v[i]);
                else row_store<false>(y_row, a.x_type, of, C, v[i]);
            }
            row_mask(of, C, v[i]);
        });
    } else {
        each([&](int i, RowVector of) { row_values(x[i], a.x_type, v[i]), row_mask(of, C, v[i]); });
    }
    if (a.out_type == CLDNN_HIP_NO_TYPE) return;
    block_norm_unit<LANES, NV, SURE>(v, a.norm, C, a.epsilon, lane, slot + 2);
    float most = 0.0f;
    each([&](int i, RowVector of) {
        float f[8];
        if (p.weight) row_floats(p.weight, of.c, C, f), times(i, f);
        if (p.bias) row_floats(p.bias, of.c, C, f), plus(i, f);
        if (p.scale) {
            modulation(p.scale, a.scale_pitch, of.c, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= 1.0f + f[j];
        }
        if (p.shift) modulation(p.shift, a.shift_pitch, of.c, f), plus(i, f);
        row_mask(of, C, v[i]);
        most = row_magnitude(v[i], most);
    });
    if (a.out_type == CLDNN_HIP_S8) {
        const RowSteps steps = row_steps(row_most<LANES>(most, slot[4]));
        each([&](int i, RowVector of) { row_store_s8((int8_t*)p.out + row * a.out_pitch, of, C, v[i], steps); });
        if (lane == 0) p.out_scales[row] = steps.scale;
    } else {
        char* out_row = (char*)p.out + row * a.out_pitch * block_norm_size(a.out_type);
        if (a.past_out) each([&](int i, RowVector of) { row_store<true>(out_row, a.out_type, of, C, v[i]); });
        else each([&](int i, RowVector of) { row_store<false>(out_row, a.out_type, of, C, v[i]); });
    }
}

// The shape for rows of C values.  A wave to a row as long as three vectors a lane hold it, then more waves (us, bf16 with gate, scale and
// shift: 20000 x 1500 54 by a wave, 60 by four; 12000 x 2048 49 and 41).
template <typename F>
static void block_norm_shape(int C, F&& f)
{
    (void)(try_row_shape<16, 1, 0>(C, f) || try_row_shape<16, 2, 1>(C, f) || try_row_shape<64, 1, 0>(C, f) || try_row_shape<64, 2, 1>(C, f) || try_row_shape<64, 3, 2>(C, f) ||
           try_row_shape<256, 1, 0>(C, f) || try_row_shape<256, 2, 1>(C, f) || try_row_shape<256, 3, 2>(C, f) || try_row_shape<512, 2, 1>(C, f) || try_row_shape<512, 3, 2>(C, f) ||
           try_row_shape<512, 4, 3>(C, f) || try_row_shape<512, 6, 4>(C, f) || try_row_shape<512, 8, 6>(C, f));
}

std::unique_ptr<OperatorPlan> block_norm_plan(const cldnn_hip_engine_s&, const cldnn_hip_block_norm_desc& d, cldnn_hip_operator_info& info)
{
    CHIP_REQUIRE(d.tokens > 0 && d.features > 0 && d.tokens_per_image >= 0, CLDNN_HIP_INVALID_ARG, "block norm: sizes must be positive");
    CHIP_REQUIRE(d.features <= ROW_MOST, CLDNN_HIP_UNSUPPORTED_SIZE, "block norm: too many features, more than 32768");
    const bool branch = d.branch_dtype != CLDNN_HIP_NO_TYPE, out = d.out_dtype != CLDNN_HIP_NO_TYPE, quantized = d.out_dtype == CLDNN_HIP_S8;
    const int64_t x_size = float_size(d.dtype, "block norm"), branch_size = branch ? float_size(d.branch_dtype, "block norm") : 0;
    const int64_t out_size = !out ? 0 : quantized ? 1 : float_size(d.out_dtype, "block norm");
    if (d.modulation_dtype != CLDNN_HIP_NO_TYPE) (void)float_size(d.modulation_dtype, "block norm");
    const auto known = [](int norm) { return norm >= CLDNN_HIP_TOKEN_NORM_NONE && norm <= CLDNN_HIP_TOKEN_NORM_RMS; };
    CHIP_REQUIRE(known(d.norm) && known(d.post), CLDNN_HIP_INVALID_ARG, "block norm: unknown norm");
    CHIP_REQUIRE(d.epsilon >= 0.0f && d.post_epsilon >= 0.0f, CLDNN_HIP_INVALID_ARG, "block norm: epsilon must not be negative");
    CHIP_REQUIRE(branch || out, CLDNN_HIP_INVALID_ARG, "block norm: neither a branch nor an output");
    CHIP_REQUIRE(branch || (d.post == CLDNN_HIP_TOKEN_NORM_NONE && d.residual_scale == 1.0f), CLDNN_HIP_INVALID_ARG, "block norm: a norm or scale of a branch without one");
    CHIP_REQUIRE(out || d.norm == CLDNN_HIP_TOKEN_NORM_NONE, CLDNN_HIP_INVALID_ARG, "block norm: a norm without an output");
    std::unique_ptr<BlockNormPlan> plan(new BlockNormPlan());
    BlockNormArgs& a = plan->a;
    a.tokens = d.tokens, a.C = d.features, a.per_image = d.tokens_per_image;
    a.x_type = d.dtype, a.branch_type = d.branch_dtype, a.out_type = d.out_dtype, a.mod_type = d.modulation_dtype;
    a.norm = d.norm, a.post = d.post, a.epsilon = d.epsilon, a.post_epsilon = d.post_epsilon, a.residual_scale = d.residual_scale;
    const auto pitch = [&](int64_t stride) {
        CHIP_REQUIRE(stride == 0 || stride >= d.features, CLDNN_HIP_INVALID_ARG, "block norm: a stride shorter than its row");
        return stride ? stride : d.features;
    };
    a.x_pitch = pitch(d.x_stride), a.branch_pitch = pitch(d.branch_stride), a.y_pitch = pitch(d.y_stride), a.out_pitch = pitch(d.out_stride);
    a.gate_pitch = pitch(d.gate_stride), a.scale_pitch = pitch(d.scale_stride), a.shift_pitch = pitch(d.shift_stride);
    block_norm_shape(d.features, [&](auto lanes, auto vectors, auto) { plan->shape = {decltype(lanes)::value, decltype(vectors)::value}; });
    const int64_t blocks = plan->shape.blocks(d.tokens);
    check_grid(blocks, plan->shape.threads(), "block norm");
    info.launches = 1, info.grid = (int32_t)blocks, info.block = plan->shape.threads(), info.lds_bytes = plan->shape.lanes > 64 ? 5 * plan->shape.lanes / 64 * 4 : 0;
    const int64_t values = d.tokens * d.features;
    info.ops = 20 * values;
    info.bytes = values * (x_size + (branch ? branch_size + x_size : 0) + out_size) + (quantized ? 4 * d.tokens : 0);
    // The stream is next read behind a whole block: it leaves the caches to what is read sooner, where all of this does not fit them.  So does
    // a result that does not fit them by itself.  (25088 x 1024 in bf16, stream / result / both past the caches: 51.2 us without, 50.6, 50.0 and
    // 43.5; the stream of 6272 x 1024 in f32 alone, with the product behind it 35.2 and 33.0.)
    a.past_y = info.bytes >= ROW_PAST, a.past_out = values * out_size >= ROW_PAST;
    snprintf(info.kernel_name, sizeof info.kernel_name, "block_norm<%dx%d>", plan->shape.lanes, plan->shape.vectors);
    return plan;
}

void block_norm_launch(hipStream_t s, const OperatorPlan& plan, const BlockNormPointers& of)
{
    const BlockNormPlan& p = static_cast<const BlockNormPlan&>(plan);
    const BlockNormArgs& a = p.a;
    BlockNormPointers given = of;
    // what the description has not is not looked at
    if (a.branch_type == CLDNN_HIP_NO_TYPE) given.branch = nullptr, given.post_weight = given.post_bias = nullptr, given.gate = nullptr, given.y = nullptr;
    if (a.out_type == CLDNN_HIP_NO_TYPE) given.out = nullptr, given.weight = given.bias = nullptr, given.scale = given.shift = nullptr;
    if (a.out_type != CLDNN_HIP_S8) given.out_scales = nullptr;
    if (a.mod_type == CLDNN_HIP_NO_TYPE) given.gate = given.scale = given.shift = nullptr;
    CHIP_REQUIRE((a.branch_type == CLDNN_HIP_NO_TYPE || given.branch) && (a.out_type == CLDNN_HIP_NO_TYPE ? given.y != nullptr : given.out != nullptr) &&
                     (a.out_type != CLDNN_HIP_S8 || given.out_scales),
                 CLDNN_HIP_INVALID_ARG, "null device pointer");
    CHIP_REQUIRE(given.y != given.x || a.y_pitch == a.x_pitch, CLDNN_HIP_INVALID_ARG, "block norm: y in the place of x with another stride");
    const int x_align = float_size(a.x_type, "");
    check_aligned(given.x, x_align, "x"), check_aligned(given.y, x_align, "y");
    if (given.branch) check_aligned(given.branch, float_size(a.branch_type, ""), "branch");
    if (given.out && a.out_type != CLDNN_HIP_S8) check_aligned(given.out, float_size(a.out_type, ""), "output");
    if (a.mod_type != CLDNN_HIP_NO_TYPE) {
        const int to = float_size(a.mod_type, "");
        check_aligned(given.gate, to, "gate"), check_aligned(given.scale, to, "scale"), check_aligned(given.shift, to, "shift");
    }
    check_aligned(given.post_weight, 4, "post_weight"), check_aligned(given.post_bias, 4, "post_bias"), check_aligned(given.weight, 4, "weight"), check_aligned(given.bias, 4, "bias");
    check_aligned(given.out_scales, 4, "out_scales");
    block_norm_shape(a.C, [&](auto lanes, auto vectors, auto sure) {
        hipLaunchKernelGGL((block_norm_kernel<decltype(lanes)::value, decltype(vectors)::value, decltype(sure)::value>), dim3((unsigned)p.shape.blocks(a.tokens)),
                           dim3(p.shape.threads()), 0, s, a, given);
    });
    CHIP_CHECK(hipGetLastError());
}

}  // namespace chip
