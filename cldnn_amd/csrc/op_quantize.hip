// Rows to int8 with a scale each: q = rint(y * (127 / max |y|)), y = act(x) * factor, or act(x) * gate * factor.
//
// A row is read once and held in registers between its maximum and its values.
#include "row_kernel.h"

namespace chip {

constexpr int QUANTIZE_FAR = 1024;  // threads to a row that registers do not hold

struct QuantizeArgs {
    int64_t rows, in_pitch, out_pitch;
    int32_t C, type, gated;
    Act act;
};

namespace {
struct QuantizePlan : OperatorPlan {
    QuantizeArgs a{};
    bool factors = false;
    RowShape shape{};  // lanes 0: rows longer than what registers hold
};
}  // namespace

__device__ __forceinline__ void quantize_values(const QuantizeArgs& a, const RowRaw& x, const RowRaw& gate, const float* factors, int c, float (&v)[8])
{
    row_values(x, a.type, v);
    act_apply<true>(v, a.act);
    if (a.gated) {
        float g[8];
        row_values(gate, a.type, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= g[i];
    }
    if (factors) {
        float f[8];
        row_floats(factors, c, a.C, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= f[i];
    }
    // what lies behind the row counts for nothing, whatever its activation
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < a.C ? v[i] : 0.0f;
}

template <int LANES, int NV>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void quantize_kernel(QuantizeArgs a, const char* in, const float* factors, int8_t* out, float* scales)
{
    constexpr int THREADS = LANES < 256 ? 256 : LANES;
    __shared__ float slot[THREADS / 64];
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t row = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) return;  // whole groups: nobody waits for them
    const int size = a.type == CLDNN_HIP_F32 ? 4 : 2;
    const char* src = in + row * a.in_pitch * size;
    RowRaw x[NV], gate[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * LANES) * 8;
        x[i] = row_load(src, a.type, c, a.C);
        if (a.gated) gate[i] = row_load(src + (int64_t)a.C * size, a.type, c, a.C);
    }
    float v[NV][8];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        quantize_values(a, x[i], gate[i], factors, (lane + i * LANES) * 8, v[i]);
        most = row_magnitude(v[i], most);
    }
    const RowSteps steps = row_steps(row_most<LANES>(most, slot));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * LANES) * 8;
        if (c < a.C) row_store_s8(out + row * a.out_pitch + c, a.C - c, v[i], steps);
    }
    if (lane == 0) scales[row] = steps.scale;
}

// Rows that registers do not hold: read twice, the second time from the caches.
__global__ __launch_bounds__(QUANTIZE_FAR) void quantize_far_kernel(QuantizeArgs a, const char* in, const float* factors, int8_t* out, float* scales)
{
    __shared__ float slot[QUANTIZE_FAR / 64];
    const int64_t row = blockIdx.x;
    const int size = a.type == CLDNN_HIP_F32 ? 4 : 2;
    const char* src = in + row * a.in_pitch * size;
    const auto each = [&](auto&& f) {
        for (int64_t c = 8 * threadIdx.x; c < a.C; c += 8 * QUANTIZE_FAR) {
            RowRaw gate{};
            const RowRaw x = row_load(src, a.type, (int)c, a.C);
            if (a.gated) gate = row_load(src + (int64_t)a.C * size, a.type, (int)c, a.C);
            float v[8];
            quantize_values(a, x, gate, factors, (int)c, v);
            f((int)c, v);
        }
    };
    uint32_t most = 0;
    each([&](int, const float (&v)[8]) { most = row_magnitude(v, most); });
    const RowSteps steps = row_steps(row_most<QUANTIZE_FAR>(most, slot));
    each([&](int c, const float (&v)[8]) { row_store_s8(out + row * a.out_pitch + c, a.C - c, v, steps); });
    if (threadIdx.x == 0) scales[row] = steps.scale;
}

std::unique_ptr<OperatorPlan> quantize_plan(const cldnn_hip_engine_s&, const cldnn_hip_quantize_desc& d, cldnn_hip_operator_info& info)
{
    CHIP_REQUIRE(d.rows > 0 && d.features > 0, CLDNN_HIP_INVALID_ARG, "quantize: sizes must be positive");
    // so that a vector's last value has a number
    CHIP_REQUIRE(d.features <= INT32_MAX / 2 - 64, CLDNN_HIP_UNSUPPORTED_SIZE, "quantize: rows too large");
    const int64_t size = float_size(d.dtype, "quantize");
    std::unique_ptr<QuantizePlan> plan(new QuantizePlan());
    QuantizeArgs& a = plan->a;
    a.rows = d.rows, a.C = d.features, a.type = d.dtype, a.gated = d.gated != 0;
    const int64_t values = (int64_t)d.features * (a.gated ? 2 : 1);
    CHIP_REQUIRE((d.in_stride == 0 || d.in_stride >= values) && (d.out_stride == 0 || d.out_stride >= d.features), CLDNN_HIP_INVALID_ARG, "quantize: a stride shorter than its row");
    a.in_pitch = d.in_stride ? d.in_stride : values, a.out_pitch = d.out_stride ? d.out_stride : d.features;
    a.act = make_act(d.activation, d.activation_m, d.activation_n, "quantize");
    plan->factors = d.has_factors != 0;
    const bool far = d.features > ROW_MOST;
    if (!far) plan->shape = row_shape(d.features);
    const int threads = far ? QUANTIZE_FAR : plan->shape.threads();
    const int64_t blocks = far ? d.rows : plan->shape.blocks(d.rows);
    check_grid(blocks, threads, "quantize");
    info.launches = 1, info.grid = (int32_t)blocks, info.block = threads, info.lds_bytes = far || plan->shape.lanes > 64 ? threads / 64 * 4 : 0;
    info.ops = 4 * d.rows * values;
    info.bytes = d.rows * (values * size + d.features + 4) + (plan->factors ? 4ll * d.features : 0);
    if (far) snprintf(info.kernel_name, sizeof info.kernel_name, "quantize_far");
    else snprintf(info.kernel_name, sizeof info.kernel_name, "quantize<%dx%d>", plan->shape.lanes, plan->shape.vectors);
    return plan;
}

void quantize_launch(hipStream_t s, const OperatorPlan& plan, const void* in, const float* factors, void* out, float* scales)
{
    const QuantizePlan& p = static_cast<const QuantizePlan&>(plan);
    const QuantizeArgs& a = p.a;
    CHIP_REQUIRE(!p.factors || factors, CLDNN_HIP_INVALID_ARG, "null device pointer");
    check_aligned(in, float_size(a.type, ""), "input"), check_aligned(scales, 4, "scales");
    if (!p.factors) factors = nullptr;
    else check_aligned(factors, 4, "factors");
    if (!p.shape.lanes) {
        hipLaunchKernelGGL(quantize_far_kernel, dim3((unsigned)a.rows), dim3(QUANTIZE_FAR), 0, s, a, (const char*)in, factors, (int8_t*)out, scales);
    } else {
        with_row_shape(p.shape, [&](auto lanes, auto vectors) {
            hipLaunchKernelGGL((quantize_kernel<decltype(lanes)::value, decltype(vectors)::value>), dim3((unsigned)p.shape.blocks(a.rows)), dim3(p.shape.threads()), 0, s, a,
                               (const char*)in, factors, (int8_t*)out, scales);
        });
    }
    CHIP_CHECK(hipGetLastError());
}

}  // namespace chip
