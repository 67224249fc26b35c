// Rotary positions with several axes.
//
// angle = position * frequency is held in turns: with frequency / (2 pi) as the sum of two floats hi + lo (worked out in 64 bits
// when the object is made), position * hi is split exactly into its rounded product and the rest, the whole turns are dropped
// from the product, and what is left is below one turn and good to about 2^-24 of a turn whatever the position.
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
    int32_t head_size;
    int32_t float_positions, inverse;
    int64_t q_pt, q_ph, k_pt, k_ph, qo_pt, qo_ph, ko_pt, ko_ph;
};

struct RotaryPlan {
    RotaryArgs a;
    int dt, pos_size, work;
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

// A thread turns one pair (or copies one value) of a token in all of its heads: one sine and cosine for all of them.
template <typename T>
__global__ __launch_bounds__(ROTARY_THREADS) void rotary_kernel(RotaryArgs a, const RotaryPair* table, const void* positions, const T* q, const T* k, T* qo, T* ko)
{
    const int work = a.pairs + a.copied;
    const int64_t i = (int64_t)blockIdx.x * ROTARY_THREADS + threadIdx.x;
    const int64_t token = i / work;
    const int w = (int)(i - token * work);
    if (token >= a.tokens) return;
    q += token * a.q_pt, qo += token * a.qo_pt;
    if (a.k_heads) k += token * a.k_pt, ko += token * a.ko_pt;
    if (w >= a.pairs) {
        const int at = a.pairs + w;
        for (int h = 0; h < a.q_heads; ++h) qo[h * a.qo_ph + at] = q[h * a.q_ph + at];
        for (int h = 0; h < a.k_heads; ++h) ko[h * a.ko_ph + at] = k[h * a.k_ph + at];
        return;
    }
    const RotaryPair p = table[w];
    const int64_t at = token * a.axes + p.axis;
    float s, c;
    rotary_turn(a.float_positions ? ((const float*)positions)[at] : (float)((const int32_t*)positions)[at], p, s, c);
    if (a.inverse) s = -s;
    const auto turn = [&](const T* x, T* y, int heads, int64_t xp, int64_t yp) {
#pragma unroll 4
        for (int h = 0; h < heads; ++h) {
            const float x0 = (float)x[h * xp + p.first], x1 = (float)x[h * xp + p.second];
            y[h * yp + p.first] = (T)(x0 * c - x1 * s);
            y[h * yp + p.second] = (T)(x1 * c + x0 * s);
        }
    };
    turn(q, qo, a.q_heads, a.q_ph, a.qo_ph);
    turn(k, ko, a.k_heads, a.k_ph, a.ko_ph);
}

RotaryPlan* rotary_plan(const cldnn_hip_engine_s&, const cldnn_hip_rotary_desc& d, cldnn_hip_operator_info& info, std::vector<char>& init)
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
    a.tokens = d.tokens, a.q_heads = d.q_heads, a.k_heads = d.k_heads, a.axes = d.axes, a.head_size = d.head_size;
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
    plan->dt = d.dtype, plan->work = a.pairs + a.copied;
    const int64_t blocks = (d.tokens * plan->work + ROTARY_THREADS - 1) / ROTARY_THREADS;
    CHIP_REQUIRE(d.tokens < (1ll << 40) && blocks < (1ll << 31), CLDNN_HIP_UNSUPPORTED_SIZE, "rotary: too many tokens");
    const int64_t n = d.tokens * (d.q_heads + d.k_heads) * d.head_size;
    info.launches = 1, info.grid = (int)blocks, info.block = ROTARY_THREADS;
    info.workspace_bytes = (int64_t)init.size();
    info.ops = 3 * n, info.bytes = 2 * n * size + 4 * d.tokens * d.axes;
    snprintf(info.kernel_name, sizeof info.kernel_name, "rotary");
    return plan.release();
}

void rotary_launch(hipStream_t s, const RotaryPlan& p, const void* workspace, const void* q, const void* k, const void* positions, void* q_out, void* k_out)
{
    const RotaryArgs& a = p.a;
    CHIP_REQUIRE(!a.k_heads || (k && k_out), CLDNN_HIP_INVALID_ARG, "null device pointer");
    const int size = float_size(p.dt, "");
    check_aligned(q, size, "q"), check_aligned(k, size, "k"), check_aligned(positions, 4, "positions");
    check_aligned(q_out, size, "q output"), check_aligned(k_out, size, "k output");
    const dim3 grid((unsigned)((a.tokens * p.work + ROTARY_THREADS - 1) / ROTARY_THREADS));
    with_float(p.dt, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((rotary_kernel<T>), grid, dim3(ROTARY_THREADS), 0, s, a, (const RotaryPair*)workspace, positions, (const T*)q, (const T*)k,
                           (T*)q_out, (T*)k_out);
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(RotaryPlan* p) { delete p; }

}  // namespace chip
