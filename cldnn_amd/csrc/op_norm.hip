// Group norm with an activation, channels last.
//
// Per image and group: mean and M2 = sum (x - mean)^2 over the group's features and the whole plane.  A thread sums its own
// pixels of a feature around a value K, the mean of its c first ones: with s1 = sum (x - K), s2 = sum (x - K)^2 over the others, n
// values in all have mean = K + s1 / n and M2 = M2 of the c + s2 - s1^2 / n.  s2 is at most n / c of the result then, which is
// what its rounding grows by; K is the first value, and moved to the mean after 8, 64 .. others, so that n / c stays below 10.  (With
// the first value all the way, one unlike the rest cost 4e-3 of M2 at 1600 pixels to a thread, and costs 2e-6 so.)
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
    int32_t fold;          // log2 of the neighbouring features that a thread's parts are of: a power of two that divides a group and a vector
    int32_t lanes;         // threads that join the parts of a group: a power of two, up to a wave
    int32_t chunk, chunks; // pixels of a workgroup; workgroups along the plane
    float per_group;       // 1 / cpg: (feature + 0.5) * per_group is its group, features being at most 6144
    int32_t whole;         // planes without gaps between rows: pixel p lies at p * px
    float epsilon;
    Act act;
};

struct NormPlan {
    NormArgs a;
    int in_dt, out_dt, vec, threads, spans, B;
    bool past; // the result goes past the caches
    bool whole; // a plane to a workgroup, in one launch; two otherwise
};

constexpr int NORM_MOST_SPAN = 6144;  // features of a workgroup: their sums lie in LDS
// Leaves 128 registers to a thread: with vectors of 8, norm_apply keeps 9 to 14 values in scratch memory and norm_whole 50 to 60.
constexpr int NORM_MOST_THREADS = 1024;
// Vectors of a plane up to which one workgroup takes it (us, one launch and two: 32 of 56x56x256 f16, 12544 vectors, 33 and 54; one
// of 64x64x320, 20480 vectors, 33 and 15).
constexpr int NORM_WHOLE = 16384;

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

template <bool NT = false, typename T, int V>
__device__ inline void norm_store(T* p, const float (&v)[V])
{
    typedef T any __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if constexpr (V == 1) *p = (T)v[0];
    else if constexpr (NT) {
        any x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)v[i];
        __builtin_nontemporal_store(x, (any*)p);
    }
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

// mean and M2 of values a vector holds
template <int V>
struct NormSums {
    float K[V], s1[V], s2[V], M2[V];
    __device__ void start(const float (&v)[V])
    {
#pragma unroll
        for (int i = 0; i < V; ++i) K[i] = v[i], s1[i] = s2[i] = M2[i] = 0.0f;
    }
    // K becomes the mean of the n values so far
    __device__ void move(int n)
    {
        const float own = 1.0f / (float)n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float m = s1[i] * own;
            K[i] += m, M2[i] += s2[i] - s1[i] * m;
            s1[i] = s2[i] = 0.0f;
        }
    }
    __device__ void add(const float (&v)[V])
    {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = v[i] - K[i];
            s1[i] += d;
            s2[i] = __builtin_fmaf(d, d, s2[i]);
        }
    }
    // neighbours of one group, 2^fold of them, are one part: parts of n values each are joined two by two
    __device__ void put(const NormArgs& a, float2* row, int c, int n)
    {
        move(n);
        float (&mean)[V] = K;
        float half = 0.5f * (float)n;
#pragma unroll
        for (int step = 1; step < V; step *= 2) {
            if (step >= 1 << a.fold) break;
#pragma unroll
            for (int i = 0; i < V; i += 2 * step) {
                const float d = mean[i + step] - mean[i];
                mean[i] = __builtin_fmaf(0.5f, d, mean[i]);
                M2[i] = __builtin_fmaf(half * d, d, M2[i] + M2[i + step]);
            }
            half *= 2.0f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if ((i & ((1 << a.fold) - 1)) == 0) row[(c + i) >> a.fold] = make_float2(mean[i], M2[i]);
    }
};

// Joins N parts of a group, `total` values: part(i, n) gives mean and M2 of part i and in n how many values those are of.  The a.lanes
// threads of the group (neighbours in a wave) call this together and all get the result.  Two passes over the parts, the first
// NORM_PARTS of a thread from registers.
constexpr int NORM_PARTS = 8;
template <typename P>
__device__ inline float2 norm_join(const NormArgs& a, int N, float total, P&& part)
{
    const int lane = threadIdx.x & (a.lanes - 1);
    float2 x[NORM_PARTS];
    float n[NORM_PARTS], unused;
    const float K = part(0, unused).x;
#pragma unroll
    for (int u = 0; u < NORM_PARTS; ++u) {
        const int i = lane + u * a.lanes;
        x[u] = make_float2(K, 0.0f), n[u] = 0.0f;
        if (i < N) x[u] = part(i, n[u]);
    }
    const auto all = [&](float v) {
        for (int i = a.lanes >> 1; i; i >>= 1) v += __shfl_xor(v, i);
        return v;
    };
    float mean = 0.0f, M2 = 0.0f;
#pragma unroll
    for (int u = 0; u < NORM_PARTS; ++u) mean = __builtin_fmaf(x[u].x - K, n[u], mean);
    for (int i = lane + NORM_PARTS * a.lanes; i < N; i += a.lanes) {
        float m;
        const float2 y = part(i, m);
        mean = __builtin_fmaf(y.x - K, m, mean);
    }
    mean = K + all(mean) / total;
#pragma unroll
    for (int u = 0; u < NORM_PARTS; ++u) {
        const float d = x[u].x - mean;
        M2 += __builtin_fmaf(n[u] * d, d, x[u].y);
    }
    for (int i = lane + NORM_PARTS * a.lanes; i < N; i += a.lanes) {
        float m;
        const float2 y = part(i, m);
        M2 += __builtin_fmaf(m * (y.x - mean), y.x - mean, y.y);
    }
    return make_float2(mean, all(M2));
}

// The parts that a workgroup's threads put into LDS, n pixels in all, group by group: then(g, its mean and M2).
template <typename F>
__device__ inline void norm_join_rows(const NormArgs& a, const float2* rows, int span, int n, F&& then)
{
    const int used = min(a.rows, n), base = n / a.rows, more = n - base * a.rows;  // row r has base pixels, the first `more` one more
    const int each = a.cpg >> a.fold, pitch = a.span >> a.fold;  // parts of a group in a row, of a row
    const float inverse = 1.0f / (float)each, values = (float)(1 << a.fold);
    for (int g = threadIdx.x / a.lanes; g < span / a.cpg; g += blockDim.x / a.lanes) {
        const float2 f = norm_join(a, used * each, (float)n * (float)a.cpg, [&](int i, float& m) {
            const int r = (int)(((float)i + 0.5f) * inverse);  // i / each: there are at most 8192
            m = (float)(base + (r < more)) * values;
            return rows[r * pitch + g * each + i - r * each];
        });
        if ((threadIdx.x & (a.lanes - 1)) == 0) then(g, f);
    }
}

__device__ inline float2 norm_scale(const NormArgs& a, float2 f)
{
    return make_float2(f.x, 1.0f / __builtin_sqrtf(f.y / ((float)a.P * (float)a.cpg) + a.epsilon));
}

// Sums over n pixels from p0 on of the workgroup's features, put into LDS as each row's parts.
template <typename TI, int V>
__device__ inline void norm_sum(const NormArgs& a, const TI* src, int span, int p0, int n, float2* rows)
{
    const int r = threadIdx.x / a.cols;
    if (r >= min(a.rows, n)) return;
    for (int c = (threadIdx.x - r * a.cols) * V; c < span; c += a.cols * V) {
        NormSums<V> sums;
        float v[V];
        norm_load<TI, V>(src + c + norm_pixel(a, a.in_py, a.in_px, p0 + r), v);
        sums.start(v);
        int p = r + a.rows, so_far = 1;
        for (int more = 8; p < n; more *= 8) {
            const int end = (int)min((int64_t)n, p + (int64_t)more * a.rows);
#pragma unroll 4
            for (; p < end; p += a.rows) {
                norm_load<TI, V>(src + c + norm_pixel(a, a.in_py, a.in_px, p0 + p), v);
                sums.add(v);
            }
            so_far += more;
            if (p < n) sums.move(so_far);
        }
        sums.put(a, rows + r * (a.span >> a.fold), c, norm_share(n, r, a.rows));
    }
}

// The result of those pixels: `ready` makes the groups' statistics (mean, 1 / deviation) that `group` points to.  A thread has four
// vectors under way beside the four that it works on; the first, and its factors, are asked for in front of the statistics.  The
// activation is chosen outside the loop: with it inside, the program that a wave runs through is long enough to be what it waits for.
template <typename TI, typename TO, int V, bool NT, typename R>
__device__ inline void norm_finish(const NormArgs& a, const TI* src, TO* dst, int span, int p0, int n, const float* scale, const float* shift, const float2* group, R&& ready)
{
    typedef TI any __attribute__((ext_vector_type(V), aligned(sizeof(TI))));
    const int r = threadIdx.x / a.cols, c0 = (threadIdx.x - r * a.cols) * V;
    const auto fetch = [&](int c, int p, any (&to)[4]) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (p + u * a.rows < n) to[u] = *(const any*)(src + c + norm_pixel(a, a.in_py, a.in_px, p0 + p + u * a.rows));
    };
    any now[4], then[4];
    float mean[V], factor[V], add[V];
    const auto ask = [&](int c) {
        fetch(c, r, now);
#pragma unroll
        for (int i = 0; i < V; ++i) factor[i] = 1.0f, add[i] = 0.0f;
        if (scale) norm_load<float, V>(scale + c, factor);  // (whole vectors: one by one these loads took 6 us)
        if (shift) norm_load<float, V>(shift + c, add);
    };
    const bool live = r < a.rows && c0 < span;
    if (live) ask(c0);
    ready();
    if (!live) return;
    const auto finish = [&](auto kind) __attribute__((always_inline)) {
        for (int c = c0; c < span; c += a.cols * V) {
            if (c != c0) ask(c);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 f = group[(int)(((float)(c + i) + 0.5f) * a.per_group)];
                mean[i] = f.x, factor[i] *= f.y;
            }
            for (int p = r; p < n; p += 4 * a.rows) {
                fetch(c, p + 4 * a.rows, then);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (p + u * a.rows < n) {
                        float v[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) v[i] = act_one<decltype(kind)::value>(__builtin_fmaf((float)now[u][i] - mean[i], factor[i], add[i]), a.act.m, a.act.n);
                        norm_store<NT, TO, V>(dst + c + norm_pixel(a, a.out_py, a.out_px, p0 + p + u * a.rows), v);
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u) now[u] = then[u];
            }
        }
    };
    act_choose(a.act.kind, finish);
}

// A plane to a workgroup: the second reading finds it in the caches.  One launch.  (7x7x2048, one image: 6.2 us, of it 4.3 the launch,
// the rest three trips to memory and the join; 32 of 56x56x256, f16: 33 us, 3.1 TB/s of one reading and one writing.  The plane held in
// registers instead takes the same time and more program.)
template <typename TI, typename TO, int V>
__global__ __launch_bounds__(NORM_MOST_THREADS) void norm_whole_kernel(NormArgs a, const TI* in, const float* scale, const float* shift, TO* out)
{
    extern __shared__ float2 lds[];
    float2* group = lds + a.rows * (a.span >> a.fold);  // behind the parts of each row of threads: the groups of the span
    const int b = blockIdx.y, first = blockIdx.z * a.span, span = min(a.span, a.C - first);
    const TI* src = in + a.in_off + b * a.in_pb + first;
    norm_sum<TI, V>(a, src, span, 0, a.P, lds);
    norm_finish<TI, TO, V, false>(a, src, out + a.out_off + b * a.out_pb + first, span, 0, a.P, scale ? scale + first : nullptr, shift ? shift + first : nullptr, group, [&]() {
        __syncthreads();
        norm_join_rows(a, lds, span, a.P, [&](int g, float2 f) { group[g] = norm_scale(a, f); });
        __syncthreads();
    });
}

// The statistics of a workgroup's pixels (16 of 224x224x64, f16: 21 us, 4.9 TB/s): part[((b * chunks + chunk) * groups + g)] = (mean, M2) of group g.
template <typename TI, int V>
__global__ __launch_bounds__(NORM_MOST_THREADS) void norm_stats_kernel(NormArgs a, const TI* in, float2* part)
{
    extern __shared__ float2 lds[];  // parts of each row of threads
    const int b = blockIdx.y, first = blockIdx.z * a.span, span = min(a.span, a.C - first);
    const int p0 = blockIdx.x * a.chunk, n = min(a.chunk, a.P - p0);
    norm_sum<TI, V>(a, in + a.in_off + b * a.in_pb + first, span, p0, n, lds);
    __syncthreads();
    norm_join_rows(a, lds, span, n, [&](int g, float2 f) { part[((int64_t)b * a.chunks + blockIdx.x) * a.groups + first / a.cpg + g] = f; });
}

// The second pass: joins the parts of the workgroup's groups and writes the result for its pixels (the same maps: 38 us, 5.4 TB/s, what
// a large copy has; the second reading is what separates both passes, 59 us, from their floor of 40).  NT: past the caches, where the
// tensors are too large for them.
template <typename TI, typename TO, int V, bool NT>
__global__ __launch_bounds__(NORM_MOST_THREADS) void norm_apply_kernel(NormArgs a, const TI* in, const float* scale, const float* shift, TO* out, const float2* part)
{
    extern __shared__ float2 lds[];  // [groups of the span] mean, 1 / deviation
    const int b = blockIdx.y, first = blockIdx.z * a.span, span = min(a.span, a.C - first);
    // the pixels that the first pass read last are the likeliest to be near
    const int p0 = (a.chunks - 1 - (int)blockIdx.x) * a.chunk, n = min(a.chunk, a.P - p0);
    norm_finish<TI, TO, V, NT>(a, in + a.in_off + b * a.in_pb + first, out + a.out_off + b * a.out_pb + first, span, p0, n, scale ? scale + first : nullptr,
                               shift ? shift + first : nullptr, lds, [&]() {
        const int lane = threadIdx.x & (a.lanes - 1);
        for (int g = threadIdx.x / a.lanes; g < span / a.cpg; g += blockDim.x / a.lanes) {
            const float2* of = part + (int64_t)b * a.chunks * a.groups + first / a.cpg + g;
            const float2 f = norm_join(a, a.chunks, (float)a.P * (float)a.cpg, [&](int i, float& m) {
                m = (float)min(a.chunk, a.P - i * a.chunk) * (float)a.cpg;
                return of[(int64_t)i * a.groups];
            });
            if (lane == 0) lds[g] = norm_scale(a, f);
        }
        __syncthreads();
    });
}

constexpr size_t NORM_MOST_LDS = 64 << 10;
static size_t norm_lds(const NormPlan& p) { return (p.a.rows * (p.a.span >> p.a.fold) + (p.whole ? p.a.span / p.a.cpg : 0)) * sizeof(float2); }

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
    plan->vec = a.C % 8 == 0 && is == 2 ? 8 : a.C % 4 == 0 ? 4 : a.C % 2 == 0 ? 2 : 1;  // 16 bytes where the features allow
    // a workgroup takes whole groups whose features fill whole vectors
    int unit = a.cpg;
    while (unit % plan->vec) unit += a.cpg;
    if (unit > NORM_MOST_SPAN) unit = a.cpg, plan->vec = 1;
    const int V = plan->vec, cus = e.props.multiProcessorCount;
    while (2 << a.fold <= V && a.cpg % (2 << a.fold) == 0) ++a.fold;
    const auto shape = [&](int span, int threads) {
        a.span = std::min(a.C, span);
        plan->threads = threads;
        plan->spans = (a.C + a.span - 1) / a.span;
        a.cols = std::min((a.span + V - 1) / V, threads);
        a.rows = threads / a.cols;
        const int in_span = a.span / a.cpg;
        a.lanes = 64;
        while (a.lanes > 1 && a.lanes * in_span > threads) a.lanes >>= 1;
    };
    a.per_group = 1.0f / (float)a.cpg;
    // A plane to a workgroup: the fewest groups that make runs of 64 bytes, and threads for four vectors each.
    int span = unit;
    while (span * is < 64 && span < a.C) span += unit;
    span = std::min(span, a.C);
    const int vectors = (span + V - 1) / V;
    plan->whole = vectors <= NORM_MOST_THREADS && (int64_t)a.P * vectors <= NORM_WHOLE;
    if (plan->whole) {
        int threads = 256;
        while (threads < NORM_MOST_THREADS && (threads < vectors || (int64_t)a.P * vectors > 4ll * threads)) threads *= 2;
        shape(span, threads);
        // (a feature to a group: its parts are the most there can be)
        while (norm_lds(*plan) > NORM_MOST_LDS && threads > vectors && threads > 256) shape(span, threads /= 2);
        a.chunk = a.P;
    } else {
        shape(std::max(unit, std::min(NORM_MOST_SPAN, NORM_MOST_THREADS * V) / unit * unit), NORM_MOST_THREADS);
        const int64_t wanted = std::max<int64_t>(1, (int64_t)cus / ((int64_t)it.b * plan->spans));
        a.chunk = (int)std::max<int64_t>((a.P + wanted - 1) / wanted, std::min(a.P, a.rows * 2));
    }
    a.chunks = (a.P + a.chunk - 1) / a.chunk;
    CHIP_REQUIRE(plan->spans <= 65535, CLDNN_HIP_UNSUPPORTED_SIZE, "group norm: too many features");
    plan->in_dt = it.dtype, plan->out_dt = ot.dtype, plan->B = it.b;
    const int64_t n = (int64_t)it.b * a.P * a.C;
    // Where input and result do not fit the memory-side cache together, the result leaves it to the input's second reading (16 of
    // 224x224x64, f16: 73 and 63 us; where they do, 16 of 112x112x64, f32, it costs 3 us of 33)
    plan->past = n * (is + os) >= 160ll << 20;
    info.launches = plan->whole ? 1 : 2;
    info.grid = a.chunks * it.b * plan->spans, info.block = plan->threads;
    info.lds_bytes = (int)norm_lds(*plan);
    if (!plan->whole) info.workspace_bytes = (int64_t)it.b * a.chunks * a.groups * (int64_t)sizeof(float2);
    info.ops = 10 * n;
    info.bytes = n * (is + os) + 8 * (int64_t)a.C;
    if (plan->whole) snprintf(info.kernel_name, sizeof info.kernel_name, "norm_whole<v%d>", V);
    else snprintf(info.kernel_name, sizeof info.kernel_name, "norm_stats<v%d> + norm_apply<v%d>", V, V);
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
        const dim3 grid(a.chunks, p.B, p.spans), block(p.threads);
        if (p.whole) {
            hipLaunchKernelGGL((norm_whole_kernel<TI, TO, V>), grid, block, norm_lds(p), s, a, (const TI*)in, scale, shift, (TO*)out);
            return;
        }
        hipLaunchKernelGGL((norm_stats_kernel<TI, V>), grid, block, norm_lds(p), s, a, (const TI*)in, part);
        const auto apply = p.past ? norm_apply_kernel<TI, TO, V, true> : norm_apply_kernel<TI, TO, V, false>;
        hipLaunchKernelGGL(apply, grid, block, a.span / a.cpg * sizeof(float2), s, a, (const TI*)in, scale, shift, (TO*)out, part);
    };
    with_float(p.in_dt, [&](auto ti) {
        with_float(p.out_dt, [&](auto to) {
            switch (p.vec) {
            case 8:
                if constexpr (sizeof(ti) == 2) both(ti, to, std::integral_constant<int, 8>());
                break;
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
