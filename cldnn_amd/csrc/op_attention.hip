// Attention in one pass over the keys with the running maximum and sum of the softmax.
//
// A wave has 32 rows: the queries of one key head, those of its sharing heads side by side.  It computes the scores transposed,
// S^T = K Q^T, so that a row of the softmax lies in the registers of two lanes (32 apart), and the result transposed as well,
// O^T = V^T P^T: the registers that S^T leaves in a lane are, as they lie, the operand that this second product wants, provided
// that V's keys are taken in the same order: in a step of 16 keys lane half h has keys 4h..4h+3 and 8+4h..8+4h+3.
// Values 16h + 4i + c of a block of 32 are put into row 8i + 4h + c of V^T, so a lane ends with 16 neighbouring values of its row.
#include <cmath>

#include "ops_common.h"

namespace chip {

struct AttentionArgs {
    int32_t q_len, kv_len, kv_heads, group, head, rows;  // rows = q_len * group
    float scale;  // without a bias times log2(e); with one the scores keep their own unit, where a bias of the lowest value is finite
    int64_t q_pb, q_pt, q_ph, k_pb, k_pt, k_ph, v_pb, v_pt, v_ph, o_pb, o_pt, o_ph, b_pb, b_ph, b_pq;
};

struct AttentionPlan {
    AttentionArgs a;
    int dt, batch, size, bias_dt, has_lengths;
};

constexpr int ATT_KEYS = 64;  // of a tile

// where 16-byte chunk c of a row of D values lies in a tile in LDS: 8 neighbouring rows have their chunks in 8 different places
template <int D>
__device__ inline int att_place(int row, int c)
{
    constexpr int C = D / 8;
    const int l = row * C + c;
    return C % 8 == 0 ? l ^ (row & 7) : l ^ ((l >> 3) & 7);
}

template <typename T, int D, typename B>
__global__ __launch_bounds__(256) void attention_kernel(AttentionArgs a, const T* q, const T* k, const T* v, const int32_t* lengths, const B* bias, T* out)
{
    typedef typename vec8<T>::type V8;
    constexpr int C = D / 8, STEPS = D / 16, BLOCKS = D / 32;
    constexpr bool BIAS = !std::is_same<B, void>::value;
    constexpr float unit = BIAS ? 1.44269504f : 1.0f;
    __shared__ v4i kt[ATT_KEYS * C], vt[ATT_KEYS * C];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int b = blockIdx.z, kh = blockIdx.y;
    const int row = min((int)(blockIdx.x * 128 + wave * 32 + col), a.rows - 1);
    const int qi = row / a.group, h = kh * a.group + row - qi * a.group;
    const int length = lengths ? min(max(lengths[b], 0), a.kv_len) : a.kv_len;
    const int chunks = a.head / 8;

    V8 qf[STEPS];
    const T* qr = q + b * a.q_pb + qi * a.q_pt + h * a.q_ph;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int c = 2 * s + half;
        qf[s] = __builtin_bit_cast(V8, c < chunks ? *(const v4i*)(qr + 8 * c) : v4i{0, 0, 0, 0});
    }
    v16f o[BLOCKS] = {};
    float most = -INFINITY, sum = 0.0f;
    const T* kb = k + b * a.k_pb + kh * a.k_ph;
    const T* vb = v + b * a.v_pb + kh * a.v_ph;
    for (int key0 = 0; key0 < length; key0 += ATT_KEYS) {
        __syncthreads();
        for (int i = threadIdx.x; i < ATT_KEYS * C; i += 256) {
            const int key = i / C, c = i - key * C;
            v4i kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
            if (key0 + key < length && c < chunks) {
                kx = *(const v4i*)(kb + (int64_t)(key0 + key) * a.k_pt + 8 * c);
                vx = *(const v4i*)(vb + (int64_t)(key0 + key) * a.v_pt + 8 * c);
            }
            kt[att_place<D>(key, c)] = kx;
            vt[att_place<D>(key, c)] = vx;
        }
        __syncthreads();
        v16f s[2] = {};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
                s[t] = mfma32(__builtin_bit_cast(V8, kt[att_place<D>(32 * t + col, 2 * i + half)]), qf[i], s[t]);
        float top = most;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = key0 + 32 * t + 8 * (i / 4) + 4 * half + i % 4;
                if constexpr (BIAS) {
                    const int64_t at = b * a.b_pb + h * a.b_ph + qi * a.b_pq + min(key, a.kv_len - 1);
                    s[t][i] = __builtin_fmaf(s[t][i], a.scale, (float)bias[at]);
                } else s[t][i] *= a.scale;
                s[t][i] = key < length ? s[t][i] : -INFINITY;
                top = fmaxf(top, s[t][i]);
            }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -INFINITY ? 0.0f : top;  // a row without a key so far
        const float fade = __builtin_amdgcn_exp2f((most - base) * unit);
        most = top;
        sum *= fade;
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] *= fade;
        V8 p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f((s[t][i] - base) * unit);
                sum += e;
                p[2 * t + i / 8][i % 8] = (T)e;
            }
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
                const int d = 32 * i + 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
                V8 x;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = 16 * st + 8 * (j / 4) + 4 * half + j % 4;
                    x[j] = ((const T*)&vt[att_place<D>(key, d / 8)])[d % 8];
                }
                o[i] = mfma32(x, p[st], o[i]);
            }
    }
    sum += __shfl_xor(sum, 32);
    if ((int)(blockIdx.x * 128 + wave * 32 + col) >= a.rows) return;
    const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* to = out + b * a.o_pb + qi * a.o_pt + h * a.o_ph;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int d = 32 * i + 16 * half + 8 * j;
            V8 x;
#pragma unroll
            for (int l = 0; l < 8; ++l) x[l] = (T)(o[i][8 * j + l] * factor);
            if (d < a.head) *(V8*)(to + d) = x;
        }
}

AttentionPlan* attention_plan(const cldnn_hip_engine_s& e, const cldnn_hip_attention_desc& d, cldnn_hip_operator_info& info)
{
    const auto is_half = [](int dt) { return dt == CLDNN_HIP_F16 || dt == CLDNN_HIP_BF16; };
    CHIP_REQUIRE(d.batch > 0 && d.q_len > 0 && d.kv_len > 0 && d.q_heads > 0 && d.kv_heads > 0 && d.head_size > 0, CLDNN_HIP_INVALID_ARG,
                 "attention: sizes must be positive");
    CHIP_REQUIRE(d.q_heads % d.kv_heads == 0, CLDNN_HIP_DIMENSION_MISMATCH, "attention: the key heads must divide the query heads");
    CHIP_REQUIRE(is_half(d.dtype), CLDNN_HIP_INVALID_ARG, "attention: data must be f16 or bf16");
    CHIP_REQUIRE(d.bias_dtype == d.dtype || d.bias_dtype == CLDNN_HIP_F32 || d.bias_dtype == CLDNN_HIP_NO_TYPE, CLDNN_HIP_INVALID_ARG,
                 "attention: the bias must be of the data's type or f32");
    CHIP_REQUIRE(d.head_size % 8 == 0 && d.head_size <= 256, CLDNN_HIP_UNSUPPORTED_SIZE, "attention: head_size must be a multiple of 8 up to 256");
    CHIP_REQUIRE(d.scale == d.scale && d.scale - d.scale == 0.0f, CLDNN_HIP_INVALID_ARG, "attention: the scale must be finite");
    std::unique_ptr<AttentionPlan> plan(new AttentionPlan{});
    AttentionArgs& a = plan->a;
    a.q_len = d.q_len, a.kv_len = d.kv_len, a.kv_heads = d.kv_heads, a.group = d.q_heads / d.kv_heads, a.head = d.head_size;
    const int64_t rows = (int64_t)d.q_len * a.group;
    CHIP_REQUIRE(rows < (1ll << 31) - 256 && d.batch <= 65535 && d.kv_heads <= 65535 && d.kv_len < (1 << 30), CLDNN_HIP_UNSUPPORTED_SIZE, "attention: too large");
    a.rows = (int32_t)rows;
    a.scale = (d.bias_dtype == CLDNN_HIP_NO_TYPE ? 1.44269504f : 1.0f) * (d.scale != 0.0f ? d.scale : 1.0f / std::sqrt((float)d.head_size));
    const auto strides = [&](int heads, int len, int64_t batch, int64_t token, int64_t head, int64_t& pb, int64_t& pt, int64_t& ph) {
        ph = head ? head : d.head_size;
        pt = token ? token : (int64_t)heads * d.head_size;
        pb = batch ? batch : pt * len;
        CHIP_REQUIRE(pb > 0 && pt > 0 && ph > 0, CLDNN_HIP_INVALID_ARG, "attention: strides must not be negative");
        CHIP_REQUIRE(pb % 8 == 0 && pt % 8 == 0 && ph % 8 == 0, CLDNN_HIP_UNSUPPORTED_FORMAT, "attention: strides must be multiples of 8 elements");
    };
    strides(d.q_heads, d.q_len, d.q_batch_stride, d.q_token_stride, d.q_head_stride, a.q_pb, a.q_pt, a.q_ph);
    strides(d.kv_heads, d.kv_len, d.k_batch_stride, d.k_token_stride, d.k_head_stride, a.k_pb, a.k_pt, a.k_ph);
    strides(d.kv_heads, d.kv_len, d.v_batch_stride, d.v_token_stride, d.v_head_stride, a.v_pb, a.v_pt, a.v_ph);
    strides(d.q_heads, d.q_len, d.out_batch_stride, d.out_token_stride, d.out_head_stride, a.o_pb, a.o_pt, a.o_ph);
    CHIP_REQUIRE(d.bias_batch_stride >= 0 && d.bias_head_stride >= 0 && d.bias_q_stride >= 0, CLDNN_HIP_INVALID_ARG, "attention: strides must not be negative");
    a.b_pb = d.bias_batch_stride, a.b_ph = d.bias_head_stride, a.b_pq = d.bias_q_stride;
    plan->dt = d.dtype, plan->batch = d.batch, plan->bias_dt = d.bias_dtype, plan->has_lengths = d.has_key_lengths != 0;
    plan->size = d.head_size <= 32 ? 32 : d.head_size <= 64 ? 64 : d.head_size <= 96 ? 96 : d.head_size <= 128 ? 128 : d.head_size <= 160 ? 160 : 256;
    const int64_t scores = (int64_t)d.batch * d.q_heads * d.q_len * d.kv_len;
    const int64_t bias_size = d.bias_dtype == CLDNN_HIP_NO_TYPE ? 0 : d.bias_dtype == CLDNN_HIP_F32 ? 4 : 2;
    info.launches = 1, info.block = 256;
    info.grid = (int)((rows + 127) / 128 * d.kv_heads * d.batch);
    info.lds_bytes = 2 * ATT_KEYS * plan->size * 2;
    info.ops = 4 * scores * d.head_size;
    info.bytes = 4ll * d.batch * d.head_size * ((int64_t)d.q_len * d.q_heads + (int64_t)d.kv_len * d.kv_heads)
                 + bias_size * (a.b_pb ? d.batch : 1) * (a.b_ph ? d.q_heads : 1) * (a.b_pq ? d.q_len : 1) * (int64_t)d.kv_len;
    snprintf(info.kernel_name, sizeof info.kernel_name, "attention<%d>", plan->size);
    return plan.release();
}

void attention_launch(hipStream_t s, const AttentionPlan& p, void* workspace, const void* q, const void* k, const void* v, const int32_t* lengths,
                      const void* bias, void* out)
{
    const AttentionArgs& a = p.a;
    const bool has_bias = p.bias_dt != CLDNN_HIP_NO_TYPE;
    CHIP_REQUIRE((!p.has_lengths || lengths) && (!has_bias || bias), CLDNN_HIP_INVALID_ARG, "null device pointer");
    check_aligned(q, 16, "q"), check_aligned(k, 16, "k"), check_aligned(v, 16, "v"), check_aligned(out, 16, "output");
    if (p.has_lengths) check_aligned(lengths, 4, "key_lengths");
    else lengths = nullptr;
    if (has_bias) check_aligned(bias, p.bias_dt == CLDNN_HIP_F32 ? 4 : 2, "bias");
    const dim3 grid((unsigned)((a.rows + 127) / 128), a.kv_heads, p.batch);
    with_half(p.dt, [&](auto t) {
        typedef decltype(t) T;
        const auto launch = [&](auto d) {
            constexpr int D = decltype(d)::value;
            const T *qt = (const T*)q, *kt = (const T*)k, *vt = (const T*)v;
            if (!has_bias) hipLaunchKernelGGL((attention_kernel<T, D, void>), grid, dim3(256), 0, s, a, qt, kt, vt, lengths, (const void*)nullptr, (T*)out);
            else if (p.bias_dt == CLDNN_HIP_F32) hipLaunchKernelGGL((attention_kernel<T, D, float>), grid, dim3(256), 0, s, a, qt, kt, vt, lengths, (const float*)bias, (T*)out);
            else hipLaunchKernelGGL((attention_kernel<T, D, T>), grid, dim3(256), 0, s, a, qt, kt, vt, lengths, (const T*)bias, (T*)out);
        };
        switch (p.size) {
        case 32: launch(std::integral_constant<int, 32>()); break;
        case 64: launch(std::integral_constant<int, 64>()); break;
        case 96: launch(std::integral_constant<int, 96>()); break;
        case 128: launch(std::integral_constant<int, 128>()); break;
        case 160: launch(std::integral_constant<int, 160>()); break;
        default: launch(std::integral_constant<int, 256>());
        }
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(AttentionPlan* p) { delete p; }

}  // namespace chip
