// Rows to int8 with a scale each: q = rint(y * (127 / max |y|)), y = act(x) * factor, or act(x) * gate * factor.
//
// A row is read once and held in registers between its maximum and its values.  25088 x 4096 in f16, 308 MB: 56 us, 5.5 TB/s of what is partly
// in the caches; behind a gelu 60 us, and 66 to 73 in turn with a large product: its 12 instructions to a value, the exponential at a quarter of
// the rate, keep the vector units as long as the rows' trips to memory take, and three waves of a SIMD overlap the two in part.
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
    bool factors = false, waves = false;
    RowShape shape{};  // lanes 0: rows longer than what registers hold
};
}  // namespace

// the values of a vector; what is not the lane's counts for nothing, whatever its activation
template <int KIND, bool WIDE>
__device__ __forceinline__ void quantize_values(const QuantizeArgs& a, const RowRaw<WIDE>& x, const RowRaw<WIDE>& gate, const float* factors, const RowVector& of, int C, float (&v)[8])
{
    row_values(x, a.type, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_one<KIND, true>(v[i], a.act.m, a.act.n);
    if (a.gated) {
        float g[8];
        row_values(gate, a.type, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= g[i];
    }
    if (factors) {
        float f[8];
        row_floats(factors, of.c, C, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= f[i];
    }
    row_mask(of, C, v);
}

template <bool WIDE, int LANES, int NV, int SURE>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES, row_waves(NV)) void quantize_kernel(QuantizeArgs a, const char* in, const float* factors, int8_t* out, float* scales)
{
    constexpr int THREADS = LANES < 256 ? 256 : LANES;
    __shared__ float slot[THREADS / 64];
    const int lane = threadIdx.x & (LANES - 1), C = row_length<LANES, SURE>(a.C);
    const int64_t row = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) return;  // whole groups: nobody waits for them
    const auto each = [&](auto&& f) __attribute__((always_inline)) { row_each<LANES, NV, SURE>(lane, C, f); };
    const int size = WIDE ? 4 : 2;
    const char* src = in + row * a.in_pitch * size;
    RowRaw<WIDE> x[NV], gate[NV];
    each([&](int i, RowVector of) { x[i] = row_load<WIDE>(src, a.type, of.c, C); });
    if (a.gated) each([&](int i, RowVector of) { gate[i] = row_load<WIDE>(src + (int64_t)C * size, a.type, of.c, C); });
    float v[NV][8], most = 0.0f;
    act_choose(a.act.kind, [&](auto kind) __attribute__((always_inline)) {
        each([&](int i, RowVector of) {
            quantize_values<decltype(kind)::value>(a, x[i], gate[i], factors, of, C, v[i]);
            most = row_magnitude(v[i], most);
        });
    });
    const RowSteps steps = row_steps(row_most<LANES>(most, slot));
    each([&](int i, RowVector of) { row_store_s8(out + row * a.out_pitch, of, C, v[i], steps); });
    if (lane == 0) scales[row] = steps.scale;
}

// Rows that registers do not hold: read twice, the second time from the caches, and their activation is worked out twice.  1000 x 40000 in f16,
// 120 MB: 34 us, 3.5 TB/s, behind a gelu 47; in f32 behind a gelu 61.  A vector of a thread is under way at a time, which the two workgroups of
// a CU cover in part.
__global__ __launch_bounds__(QUANTIZE_FAR) void quantize_far_kernel(QuantizeArgs a, const char* in, const float* factors, int8_t* out, float* scales)
{
    __shared__ float slot[QUANTIZE_FAR / 64];
    const int64_t row = blockIdx.x;
    const int size = a.type == CLDNN_HIP_F32 ? 4 : 2;
    const char* src = in + row * a.in_pitch * size;
    act_choose(a.act.kind, [&](auto kind) __attribute__((always_inline)) {
        const auto each = [&](auto&& f) {
            for (int64_t c = 8 * threadIdx.x; c < a.C; c += 8 * QUANTIZE_FAR) {
                const int at = (int)min(c, (int64_t)a.C - 8);
                const RowVector of{at, (int)c - at};
                RowRaw<true> gate{};
                const RowRaw<true> x = row_load<true>(src, a.type, at, a.C);
                if (a.gated) gate = row_load<true>(src + (int64_t)a.C * size, a.type, at, a.C);
                float v[8];
                quantize_values<decltype(kind)::value>(a, x, gate, factors, of, a.C, v);
                f(of, v);
            }
        };
        float most = 0.0f;
        each([&](const RowVector&, const float (&v)[8]) { most = row_magnitude(v, most); });
        const RowSteps steps = row_steps(row_most<QUANTIZE_FAR>(most, slot));
        each([&](const RowVector& of, const float (&v)[8]) { row_store_s8(out + row * a.out_pitch, of, a.C, v, steps); });
        if (threadIdx.x == 0) scales[row] = steps.scale;
    });
}

// The shape for rows of C values.  waves: there are enough rows of a 16-bit type for a wave to each, up to 8 vectors a lane, which pays the
// row's maximum and quotients once for more values (us, f16 with a gelu, by a wave and by four: 25088 x 4096 73 and 78, 25088 x 3000 42 and
// 56; 1000 x 4096 5.8 and 5.1).
template <typename F>
static void quantize_shape(int C, bool waves, F&& f)
{
    (void)(try_row_shape<16, 1, 0>(C, f) || try_row_shape<16, 2, 1>(C, f) || try_row_shape<64, 1, 0>(C, f) || try_row_shape<64, 2, 1>(C, f) || try_row_shape<64, 3, 2>(C, f) ||
           try_row_shape<64, 4, 3>(C, f) || (waves && (try_row_shape<64, 6, 4>(C, f) || try_row_shape<64, 8, 6>(C, f))) || try_row_shape<256, 2, 1>(C, f) ||
           try_row_shape<256, 3, 2>(C, f) || try_row_shape<512, 2, 1>(C, f) || try_row_shape<512, 3, 2>(C, f) || try_row_shape<512, 4, 3>(C, f) || try_row_shape<512, 6, 4>(C, f) ||
           try_row_shape<512, 8, 6>(C, f));
}

std::unique_ptr<OperatorPlan> quantize_plan(const cldnn_hip_engine_s& e, const cldnn_hip_quantize_desc& d, cldnn_hip_operator_info& info)
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
    plan->waves = size == 2 && d.rows >= 16ll * e.props.multiProcessorCount;
    if (!far) quantize_shape(d.features, plan->waves, [&](auto lanes, auto vectors, auto) { plan->shape = {decltype(lanes)::value, decltype(vectors)::value}; });
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
        quantize_shape(a.C, p.waves, [&](auto lanes, auto vectors, auto sure) {
            constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value, S = decltype(sure)::value;
            auto kernel = quantize_kernel<false, L, V, S>;
            if constexpr (L != 64 || V <= 4) kernel = a.type == CLDNN_HIP_F32 ? quantize_kernel<true, L, V, S> : kernel;
            hipLaunchKernelGGL(kernel, dim3((unsigned)p.shape.blocks(a.rows)), dim3(p.shape.threads()), 0, s, a, (const char*)in, factors, (int8_t*)out, scales);
        });
    }
    CHIP_CHECK(hipGetLastError());
}

}  // namespace chip
