// Rotary positions with several axes.
//
// angle = position * frequency is held in turns: with frequency / (2 pi) as the sum of two floats hi + lo (worked out in 64 bits
// when the object is made), position * hi is split exactly into its rounded product and the rest, the whole turns are dropped
// from the product, and what is left is below one turn and good to about 2^-24 of a turn as long as position * frequency is below
// 2^24: for every position that a float has exactly, where the base is 1 or more.  (Beyond, the rest is whole turns itself, and the
// frequency's own 48 bits are too few: position 2^24, base 1e-4: 2^-13 of a turn.)
#include <cmath>

#include "ops_common.h"

namespace chip {

// one pair of a head, as the table in the object's memory has it
struct RotaryPair {
    float hi, lo;          // frequency in turns
    int32_t axis;
    int32_t first, second; // where its two values lie
};

struct RotaryArgs {
    int64_t tokens;
    int32_t q_heads, k_heads, pairs, axes, copied;  // values behind the pairs, copied
    int32_t items;      // threads of a token and its group of heads: W pairs each, then 8 of the copied values each
    int32_t heads;      // of a group
    int32_t interleaved;
    int32_t float_positions, inverse;
    int64_t q_pt, q_ph, k_pt, k_ph, qo_pt, qo_ph, ko_pt, ko_ph;
};

struct RotaryPlan {
    RotaryArgs a;
    int dt, width, groups;
};

constexpr int ROTARY_THREADS = 256;

__device__ inline void rotary_turn(float position, const RotaryPair& p, float& s, float& c)
{
#pragma clang fp contract(off)  // the product has to be the rounded one wherever it is used
    const float product = position * p.hi;
    const float rest = __builtin_fmaf(position, p.hi, -product) + position * p.lo;
    const float turns = (product - __builtin_rintf(product)) + rest;
    sincospif(2.0f * turns, &s, &c);
}

template <typename T, int N>
struct RotaryVector {
    typedef T any __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    any v;
    __device__ void load(const T* p) { v = *(const any*)p; }
    __device__ void store(T* p) const { *(any*)p = v; }
};

// A thread turns W neighbouring pairs of a token in a group of its heads, queries' first, keys' behind them: one sine and cosine
// for all of them, worked out while the first heads' values are on their way.  Their values are two runs of W, or where pairs are
// interleaved one of 2 W.  Bound by memory: 25088 tokens with 16 + 4 heads of 128 (f16) 58 us, 4.4 TB/s where a large copy has 5.2
// (a value at a time 80 us); in halves 63 us.  196 tokens with 16 + 16 heads of 64: 4.3 us, the launch.
template <typename T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(ROTARY_THREADS) void rotary_kernel(RotaryArgs a, const RotaryPair* table, const void* positions, const T* q, const T* k, T* qo, T* ko)
{
    constexpr int AT_ONCE = 4;
    const int64_t i = (int64_t)blockIdx.x * ROTARY_THREADS + threadIdx.x;
    const int64_t token = i / a.items;
    const int w = (int)(i - token * a.items);
    if (token >= a.tokens) return;
    const int from = blockIdx.y * a.heads, to = min(from + a.heads, a.q_heads + a.k_heads);
    const auto source = [&](int h) { return h < a.q_heads ? q + token * a.q_pt + h * a.q_ph : k + token * a.k_pt + (h - a.q_heads) * a.k_ph; };
    const auto target = [&](int h) { return h < a.q_heads ? qo + token * a.qo_pt + h * a.qo_ph : ko + token * a.ko_pt + (h - a.q_heads) * a.ko_ph; };
    if (w * W >= a.pairs) {
        const int at = 2 * a.pairs + (w - a.pairs / W) * 8, n = min(8, 2 * a.pairs + a.copied - at);
        for (int h = from; h < to; ++h)
            for (int j = 0; j < n; ++j) target(h)[at + j] = source(h)[at + j];
        return;
    }
    typedef RotaryVector<T, INTERLEAVED ? 2 * W : W> Run;
    RotaryPair p[W];
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = table[w * W + j];
    float s[W], c[W], position[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const int64_t at = token * a.axes + p[j].axis;
        position[j] = a.float_positions ? ((const float*)positions)[at] : (float)((const int32_t*)positions)[at];
    }
    for (int h = from; h < to; h += AT_ONCE) {
        Run x[AT_ONCE], y[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (h + u < to) {
                x[u].load(source(h + u) + p[0].first);
                if constexpr (!INTERLEAVED) y[u].load(source(h + u) + p[0].second);
            }
        if (h == from)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                rotary_turn(position[j], p[j], s[j], c[j]);
                if (a.inverse) s[j] = -s[j];
            }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (h + u < to) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float x0 = (float)x[u].v[INTERLEAVED ? 2 * j : j], x1 = (float)(INTERLEAVED ? x[u].v[(2 * j + 1) % (2 * W)] : y[u].v[j]);
                    const T y0 = (T)(x0 * c[j] - x1 * s[j]), y1 = (T)(x1 * c[j] + x0 * s[j]);
                    if constexpr (INTERLEAVED) x[u].v[2 * j] = y0, x[u].v[2 * j + 1] = y1;
                    else x[u].v[j] = y0, y[u].v[j] = y1;
                }
                x[u].store(target(h + u) + p[0].first);
                if constexpr (!INTERLEAVED) y[u].store(target(h + u) + p[0].second);
            }
    }
}

RotaryPlan* rotary_plan(const cldnn_hip_engine_s& e, const cldnn_hip_rotary_desc& d, cldnn_hip_operator_info& info, std::vector<char>& init)
{
    const int size = float_size(d.dtype, "rotary");
    CHIP_REQUIRE(d.tokens > 0 && d.q_heads > 0 && d.k_heads >= 0 && d.head_size > 0, CLDNN_HIP_INVALID_ARG, "rotary: sizes must be positive");
    CHIP_REQUIRE(d.axes > 0 && d.axes <= CLDNN_HIP_ROTARY_MAX_AXES, CLDNN_HIP_INVALID_ARG, "rotary: one to four axes");
    CHIP_REQUIRE(d.pairing >= CLDNN_HIP_ROTARY_INTERLEAVED && d.pairing <= CLDNN_HIP_ROTARY_HALVES_PER_AXIS, CLDNN_HIP_INVALID_ARG, "rotary: unknown pairing");
    CHIP_REQUIRE(d.position_dtype == CLDNN_HIP_I32 || d.position_dtype == CLDNN_HIP_F32, CLDNN_HIP_INVALID_ARG, "rotary: positions must be i32 or f32");
    CHIP_REQUIRE(d.base > 0.0f && std::isfinite(d.base), CLDNN_HIP_INVALID_ARG, "rotary: the base must be positive");
    int64_t pairs = 0;
    for (int i = 0; i < d.axes; ++i) {
        CHIP_REQUIRE(d.pairs[i] >= 0, CLDNN_HIP_INVALID_ARG, "rotary: negative number of pairs");
        pairs += d.pairs[i];
    }
    CHIP_REQUIRE(pairs > 0 && 2 * pairs <= d.head_size, CLDNN_HIP_DIMENSION_MISMATCH, "rotary: the axes' pairs must be some, and fit the head");
    std::unique_ptr<RotaryPlan> plan(new RotaryPlan{});
    RotaryArgs& a = plan->a;
    a.tokens = d.tokens, a.q_heads = d.q_heads, a.k_heads = d.k_heads, a.axes = d.axes, a.interleaved = d.pairing == CLDNN_HIP_ROTARY_INTERLEAVED;
    a.pairs = (int)pairs, a.copied = d.head_size - 2 * (int)pairs;
    a.float_positions = d.position_dtype == CLDNN_HIP_F32, a.inverse = d.inverse != 0;
    const auto strides = [&](int heads, int64_t token, int64_t head, int64_t& pt, int64_t& ph) {
        ph = head ? head : d.head_size;
        pt = token ? token : (int64_t)heads * d.head_size;
        CHIP_REQUIRE(pt > 0 && ph > 0, CLDNN_HIP_INVALID_ARG, "rotary: strides must not be negative");
    };
    strides(d.q_heads, d.q_token_stride, d.q_head_stride, a.q_pt, a.q_ph);
    strides(d.k_heads ? d.k_heads : 1, d.k_token_stride, d.k_head_stride, a.k_pt, a.k_ph);
    strides(d.q_heads, d.q_out_token_stride, d.q_out_head_stride, a.qo_pt, a.qo_ph);
    strides(d.k_heads ? d.k_heads : 1, d.k_out_token_stride, d.k_out_head_stride, a.ko_pt, a.ko_ph);
    init.resize(pairs * sizeof(RotaryPair));
    RotaryPair* table = (RotaryPair*)init.data();
    int start = 0;
    for (int axis = 0; axis < d.axes; ++axis) {
        for (int j = 0; j < d.pairs[axis]; ++j) {
            const int i = start + j;
            const double exponent = d.shared_frequencies ? (double)i / (double)pairs : (double)j / d.pairs[axis];
            const double turns = std::pow((double)d.base, -exponent) / (2 * M_PI);
            RotaryPair& p = table[i];
            p.hi = (float)turns, p.lo = (float)(turns - (double)p.hi), p.axis = axis;
            if (d.pairing == CLDNN_HIP_ROTARY_INTERLEAVED) p.first = 2 * i, p.second = 2 * i + 1;
            else if (d.pairing == CLDNN_HIP_ROTARY_HALVES) p.first = i, p.second = i + (int)pairs;
            else p.first = 2 * start + j, p.second = 2 * start + j + d.pairs[axis];
        }
        start += d.pairs[axis];
    }
    plan->dt = d.dtype;
    // 16 bytes to a run where the pairs can be taken so, by halves of it otherwise; a run stays within an axis where that sets its place
    plan->width = 16 / size / (a.interleaved ? 2 : 1);
    const auto fits = [&](int w) {
        if (d.pairing == CLDNN_HIP_ROTARY_HALVES_PER_AXIS)
            for (int i = 0; i < d.axes; ++i)
                if (d.pairs[i] % w) return false;
        return pairs % w == 0;
    };
    while (!fits(plan->width)) plan->width /= 2;
    a.items = a.pairs / plan->width + (a.copied + 7) / 8;
    CHIP_REQUIRE(d.tokens < (1ll << 32), CLDNN_HIP_UNSUPPORTED_SIZE, "rotary: too many tokens");
    const int64_t blocks = (d.tokens * a.items + ROTARY_THREADS - 1) / ROTARY_THREADS;
    check_grid(blocks, ROTARY_THREADS, "rotary");
    CHIP_REQUIRE(std::max(d.q_heads, d.k_heads) < (1 << 29), CLDNN_HIP_UNSUPPORTED_SIZE, "rotary: too many heads");
    // heads in groups where threads are few: four waves to a SIMD before a thread takes a second group of four
    const int heads = d.q_heads + d.k_heads;
    const int64_t wanted = std::max<int64_t>(1, 4ll * e.props.multiProcessorCount / blocks);
    a.heads = (int)((heads + wanted - 1) / wanted);
    plan->groups = (heads + a.heads - 1) / a.heads;
    CHIP_REQUIRE(plan->groups <= 65535, CLDNN_HIP_UNSUPPORTED_SIZE, "rotary: too many heads");
    const int64_t n = d.tokens * (d.q_heads + d.k_heads) * d.head_size;
    info.launches = 1, info.grid = (int)blocks * plan->groups, info.block = ROTARY_THREADS;
    info.workspace_bytes = (int64_t)init.size();
    info.ops = 3 * n, info.bytes = 2 * n * size + 4 * d.tokens * d.axes;
    snprintf(info.kernel_name, sizeof info.kernel_name, "rotary<%d%s>", plan->width, a.interleaved ? ",interleaved" : "");
    return plan.release();
}

void rotary_launch(hipStream_t s, const RotaryPlan& p, const void* workspace, const void* q, const void* k, const void* positions, void* q_out, void* k_out)
{
    const RotaryArgs& a = p.a;
    CHIP_REQUIRE(!a.k_heads || (k && k_out), CLDNN_HIP_INVALID_ARG, "null device pointer");
    const int size = float_size(p.dt, "");
    check_aligned(q, size, "q"), check_aligned(k, size, "k"), check_aligned(positions, 4, "positions");
    check_aligned(q_out, size, "q output"), check_aligned(k_out, size, "k output");
    const dim3 grid((unsigned)((a.tokens * a.items + ROTARY_THREADS - 1) / ROTARY_THREADS), p.groups);
    with_float(p.dt, [&](auto t) {
        typedef decltype(t) T;
        const auto launch = [&](auto w) {
            constexpr int W = decltype(w)::value;
            const auto go = [&](auto f) {
                hipLaunchKernelGGL(f, grid, dim3(ROTARY_THREADS), 0, s, a, (const RotaryPair*)workspace, positions, (const T*)q, (const T*)k, (T*)q_out, (T*)k_out);
            };
            if (!a.interleaved) {
                if constexpr (W * sizeof(T) <= 16) go(rotary_kernel<T, W, false>);
            } else if constexpr (2 * W * sizeof(T) <= 16) go(rotary_kernel<T, W, true>);
        };
        switch (p.width) {
        case 8: launch(std::integral_constant<int, 8>()); break;
        case 4: launch(std::integral_constant<int, 4>()); break;
        case 2: launch(std::integral_constant<int, 2>()); break;
        default: launch(std::integral_constant<int, 1>());
        }
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(RotaryPlan* p) { delete p; }

}  // namespace chip
