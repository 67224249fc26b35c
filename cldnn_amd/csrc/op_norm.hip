// Group norm with an activation, channels last.
//
// Per image and group: mean and M2 = sum (x - mean)^2 over the group's features and the whole plane.  A thread sums its own few
// pixels of a feature around the first of them, K: with s1 = sum (x - K), s2 = sum (x - K)^2 over n values, mean = K + s1 / n and
// M2 = s2 - s1^2 / n, where K being one of the values bounds s2 / M2 by n (a K shared by a workgroup's rows made that hundreds).
// Parts are joined by M2 = sum M2_i + sum n_i (mean_i - mean)^2 (Chan, Golub and LeVeque), in an order that the shapes alone fix.
#include "ops_common.h"

namespace chip {

struct NormArgs {
    int64_t in_off, in_pb, in_py, in_px;   // elements; a pixel's features lie side by side
    int64_t out_off, out_pb, out_py, out_px;
    int32_t C, cpg, groups;
    int32_t W, P;          // width and size of the plane
    int32_t span;          // features of a workgroup: whole groups
    int32_t cols, rows;    // vectors across the features, pixels at a time
    int32_t chunk, chunks; // pixels of a workgroup of the statistics pass; workgroups along the plane
    int32_t chunk2;        // pixels of a workgroup of the second pass
    int32_t whole;         // planes without gaps between rows: pixel p lies at p * px
    float epsilon;
    Act act;
};

struct NormPlan {
    NormArgs a;
    int in_dt, out_dt, vec;
    int blocks2;
    int spans;
    int B;
};

constexpr int NORM_THREADS = 256;
constexpr int NORM_MOST_SPAN = 6144;  // features of a workgroup: their sums lie in LDS

template <typename T, int V>
__device__ inline void norm_load(const T* p, float (&v)[V])
{
    typedef T any __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if constexpr (V == 1) v[0] = (float)*p;
    else {
        const any x = *(const any*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)x[i];
    }
}

template <typename T, int V>
__device__ inline void norm_store(T* p, const float (&v)[V])
{
    typedef T any __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if constexpr (V == 1) *p = (T)v[0];
    else {
        any x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)v[i];
        *(any*)p = x;
    }
}

__device__ inline int64_t norm_pixel(const NormArgs& a, int64_t py, int64_t px, int p)
{
    if (a.whole) return (int64_t)p * px;
    const int y = p / a.W;
    return (int64_t)y * py + (int64_t)(p - y * a.W) * px;
}

// pixels of row r when n are dealt to `rows` of them in turn
__device__ inline int norm_share(int n, int r, int rows) { return (n - r + rows - 1) / rows; }

// The statistics of a workgroup's part: part[((b * chunks + chunk) * groups + g)] = (mean, M2) of group g.
template <typename TI, int V>
__global__ __launch_bounds__(NORM_THREADS) void norm_stats_kernel(NormArgs a, const TI* in, float2* part)
{
    extern __shared__ float2 lds[];
    float2* feature = lds;              // [span] mean, M2 of each feature
    float2* row = lds + a.span;         // [rows][cols * V] sums of each row of threads
    const int b = blockIdx.y, first = blockIdx.z * a.span, t = threadIdx.x;
    const int span = min(a.span, a.C - first);
    const int p0 = blockIdx.x * a.chunk, n = min(a.chunk, a.P - p0);
    const TI* base = in + a.in_off + b * a.in_pb + first;
    const int r = t / a.cols;
    for (int c0 = 0; c0 < span; c0 += a.cols * V) {
        const int width = min(a.cols * V, span - c0), c = (t - r * a.cols) * V;
        const bool live = r < min(a.rows, n) && c < width;
        if (live) {
            const TI* at = base + c0 + c;
            float K[V], s1[V], s2[V];
            norm_load<TI, V>(at + norm_pixel(a, a.in_py, a.in_px, p0 + r), K);
#pragma unroll
            for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
#pragma unroll 4
            for (int p = r + a.rows; p < n; p += a.rows) {
                float v[V];
                norm_load<TI, V>(at + norm_pixel(a, a.in_py, a.in_px, p0 + p), v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = v[i] - K[i];
                    s1[i] += d;
                    s2[i] = __builtin_fmaf(d, d, s2[i]);
                }
            }
            const float own = 1.0f / (float)norm_share(n, r, a.rows);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float m = s1[i] * own;
                row[r * a.cols * V + c + i] = make_float2(K[i] + m, s2[i] - s1[i] * m);
            }
        }
        __syncthreads();
        for (int f = t; f < width; f += NORM_THREADS) {
            const float K = row[f].x;
            float mean = 0.0f, M2 = 0.0f;
            for (int j = 0; j < min(a.rows, n); ++j) mean += (row[j * a.cols * V + f].x - K) * (float)norm_share(n, j, a.rows);
            mean = K + mean / (float)n;
            for (int j = 0; j < min(a.rows, n); ++j) {
                const float2 s = row[j * a.cols * V + f];
                const float d = s.x - mean;
                M2 += s.y + (float)norm_share(n, j, a.rows) * d * d;
            }
            feature[c0 + f] = make_float2(mean, M2);
        }
        __syncthreads();
    }
    for (int g = t; g < span / a.cpg; g += NORM_THREADS) {
        float mean = 0.0f, M2 = 0.0f;
        const float K = feature[g * a.cpg].x;
        for (int i = 0; i < a.cpg; ++i) mean += feature[g * a.cpg + i].x - K;
        mean = K + mean / (float)a.cpg;
        for (int i = 0; i < a.cpg; ++i) {
            const float2 f = feature[g * a.cpg + i];
            const float d = f.x - mean;
            M2 += f.y + (float)n * d * d;
        }
        part[((int64_t)b * a.chunks + blockIdx.x) * a.groups + first / a.cpg + g] = make_float2(mean, M2);
    }
}

// The second pass: joins the parts of the workgroup's groups and writes the result for its pixels.
template <typename TI, typename TO, int V>
__global__ __launch_bounds__(NORM_THREADS) void norm_apply_kernel(NormArgs a, const TI* in, const float* scale, const float* shift, TO* out, const float2* part)
{
    extern __shared__ float2 lds[];  // [groups of the span] mean, 1 / deviation
    const int b = blockIdx.y, first = blockIdx.z * a.span, t = threadIdx.x;
    const int span = min(a.span, a.C - first);
    for (int g = t; g < span / a.cpg; g += NORM_THREADS) {
        const float2* of = part + (int64_t)b * a.chunks * a.groups + first / a.cpg + g;
        const float K = of[0].x;
        float mean = 0.0f, M2 = 0.0f;
        for (int k = 0; k < a.chunks; ++k) mean += (of[(int64_t)k * a.groups].x - K) * (float)min(a.chunk, a.P - k * a.chunk);
        mean = K + mean / (float)a.P;
        for (int k = 0; k < a.chunks; ++k) {
            const float2 f = of[(int64_t)k * a.groups];
            const float d = f.x - mean;
            M2 += f.y + (float)min(a.chunk, a.P - k * a.chunk) * (float)a.cpg * d * d;
        }
        const float variance = M2 / ((float)a.P * (float)a.cpg);
        lds[g] = make_float2(mean, 1.0f / __builtin_sqrtf(variance + a.epsilon));
    }
    __syncthreads();
    const int p0 = blockIdx.x * a.chunk2, n = min(a.chunk2, a.P - p0), r = t / a.cols;
    if (r >= a.rows) return;
    const TI* src = in + a.in_off + b * a.in_pb + first;
    TO* dst = out + a.out_off + b * a.out_pb + first;
    for (int c = (t - r * a.cols) * V; c < span; c += a.cols * V) {
        float mean[V], factor[V], add[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 f = lds[(c + i) / a.cpg];
            mean[i] = f.x;
            factor[i] = scale ? f.y * scale[first + c + i] : f.y;
            add[i] = shift ? shift[first + c + i] : 0.0f;
        }
#pragma unroll 4
        for (int p = r; p < n; p += a.rows) {
            float v[V];
            norm_load<TI, V>(src + c + norm_pixel(a, a.in_py, a.in_px, p0 + p), v);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __builtin_fmaf(v[i] - mean[i], factor[i], add[i]);
            act_apply(v, a.act);
            norm_store<TO, V>(dst + c + norm_pixel(a, a.out_py, a.out_px, p0 + p), v);
        }
    }
}

NormPlan* norm_plan(const cldnn_hip_engine_s& e, const cldnn_hip_group_norm_desc& d, cldnn_hip_operator_info& info)
{
    const cldnn_hip_tensor &it = d.input, &ot = d.output;
    const int is = float_size(it.dtype, "group norm"), os = float_size(ot.dtype, "group norm");
    CHIP_REQUIRE(it.format == CLDNN_HIP_FMT_BYXF && ot.format == CLDNN_HIP_FMT_BYXF, CLDNN_HIP_UNSUPPORTED_FORMAT, "group norm: tensors must be byxf");
    CHIP_REQUIRE(it.b == ot.b && it.f == ot.f && it.y == ot.y && it.x == ot.x, CLDNN_HIP_DIMENSION_MISMATCH, "group norm keeps the sizes");
    const Pitch ip = make_pitch(it), op = make_pitch(ot);
    CHIP_REQUIRE(d.groups > 0 && it.f % d.groups == 0, CLDNN_HIP_INVALID_ARG, "group norm: groups must divide the features");
    CHIP_REQUIRE(d.epsilon >= 0.0f, CLDNN_HIP_INVALID_ARG, "group norm: epsilon must not be negative");
    CHIP_REQUIRE((int64_t)it.y * it.x < (1ll << 31) - (1 << 20), CLDNN_HIP_UNSUPPORTED_SIZE, "group norm: plane too large");
    CHIP_REQUIRE(it.b <= 65535, CLDNN_HIP_UNSUPPORTED_SIZE, "group norm: more than 65535 images");
    const Act act = make_act(d.activation, d.activation_m, d.activation_n, "group norm");
    std::unique_ptr<NormPlan> plan(new NormPlan{});
    NormArgs& a = plan->a;
    a.in_off = ip.off, a.in_pb = ip.pb, a.in_py = ip.py, a.in_px = ip.px;
    a.out_off = op.off, a.out_pb = op.pb, a.out_py = op.py, a.out_px = op.px;
    a.C = it.f, a.groups = d.groups, a.cpg = it.f / d.groups, a.W = it.x, a.P = it.y * it.x;
    a.whole = ip.py == ip.px * it.x && op.py == op.px * it.x;
    a.epsilon = d.epsilon, a.act = act;
    CHIP_REQUIRE(a.cpg <= NORM_MOST_SPAN, CLDNN_HIP_UNSUPPORTED_SIZE, "group norm: more than 6144 features in a group");
    plan->vec = a.C % 8 == 0 ? 8 : a.C % 4 == 0 ? 4 : a.C % 2 == 0 ? 2 : 1;
    // a workgroup takes whole groups whose features fill whole vectors
    int unit = a.cpg;
    while (unit % plan->vec) unit += a.cpg;
    if (unit > NORM_MOST_SPAN) unit = a.cpg, plan->vec = 1;
    const int most = std::min(NORM_MOST_SPAN, std::max(unit, NORM_THREADS * plan->vec / unit * unit));
    a.span = std::min(a.C, most / unit * unit);
    plan->spans = (a.C + a.span - 1) / a.span;
    CHIP_REQUIRE(plan->spans <= 65535, CLDNN_HIP_UNSUPPORTED_SIZE, "group norm: too many features");
    a.cols = std::min(a.span / plan->vec, NORM_THREADS);
    a.rows = NORM_THREADS / a.cols;
    const int cus = e.props.multiProcessorCount;
    const int64_t wanted = std::max<int64_t>(1, (int64_t)cus * 4 / ((int64_t)it.b * plan->spans));
    a.chunk = (int)std::max<int64_t>((a.P + wanted - 1) / wanted, std::min(a.P, a.rows * 4));
    a.chunks = (a.P + a.chunk - 1) / a.chunk;
    a.chunk2 = (int)std::max<int64_t>((a.P + 2 * wanted - 1) / (2 * wanted), std::min(a.P, a.rows * 4));
    plan->blocks2 = (a.P + a.chunk2 - 1) / a.chunk2;
    plan->in_dt = it.dtype, plan->out_dt = ot.dtype, plan->B = it.b;
    const int64_t n = (int64_t)it.b * a.P * a.C;
    info.launches = 2;
    info.grid = a.chunks * it.b * plan->spans, info.block = NORM_THREADS;
    info.lds_bytes = (int)((a.span + a.rows * a.cols * plan->vec) * sizeof(float2));
    info.workspace_bytes = (int64_t)it.b * a.chunks * a.groups * (int64_t)sizeof(float2);
    info.ops = 10 * n;
    info.bytes = n * (is + os) + 8 * (int64_t)a.C;
    snprintf(info.kernel_name, sizeof info.kernel_name, "norm_stats<v%d> + norm_apply<v%d>", plan->vec, plan->vec);
    return plan.release();
}

void norm_launch(hipStream_t s, const NormPlan& p, void* workspace, const void* in, const float* scale, const float* shift, void* out)
{
    check_aligned(in, float_size(p.in_dt, ""), "input"), check_aligned(out, float_size(p.out_dt, ""), "output");
    check_aligned(scale, 4, "scale"), check_aligned(shift, 4, "shift");
    const NormArgs& a = p.a;
    float2* part = (float2*)workspace;
    const auto both = [&](auto ti, auto to, auto v) {
        typedef decltype(ti) TI;
        typedef decltype(to) TO;
        constexpr int V = decltype(v)::value;
        const size_t lds = (a.span + a.rows * a.cols * V) * sizeof(float2);
        hipLaunchKernelGGL((norm_stats_kernel<TI, V>), dim3(a.chunks, p.B, p.spans), dim3(NORM_THREADS), lds, s, a, (const TI*)in, part);
        hipLaunchKernelGGL((norm_apply_kernel<TI, TO, V>), dim3(p.blocks2, p.B, p.spans), dim3(NORM_THREADS), a.span / a.cpg * sizeof(float2), s, a,
                           (const TI*)in, scale, shift, (TO*)out, part);
    };
    with_float(p.in_dt, [&](auto ti) {
        with_float(p.out_dt, [&](auto to) {
            switch (p.vec) {
            case 8: both(ti, to, std::integral_constant<int, 8>()); break;
            case 4: both(ti, to, std::integral_constant<int, 4>()); break;
            case 2: both(ti, to, std::integral_constant<int, 2>()); break;
            default: both(ti, to, std::integral_constant<int, 1>());
            }
        });
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(NormPlan* p) { delete p; }

}  // namespace chip
