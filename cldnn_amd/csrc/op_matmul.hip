// Matrix product with bias, activation and residual: out = act2(act(a w^T + bias) + residual).
//
// The weights are the row operand of the matrix instruction.  Its result gives a lane the values of rows 8i + 4h + c (i, c = 0..3,
// h = the lane's half) of one column; feature 16h + 4i + c of a block of 32 is put into that row, so a lane ends with 16
// neighbouring features of one row of the result: whole 16-byte stores, and a bias and a residual that are read the same way.
#include "ops_common.h"

namespace chip {

struct MatmulArgs {
    int32_t m, n, k;
    int64_t a_pitch, w_pitch, o_pitch, r_pitch;
    const float* bias;
    const void* residual;  // nullptr: none
    Act act, act2;
    int32_t res_float, out_float;
};

struct MatmulPlan {
    MatmulArgs a;
    int dt;
};

// the feature, within a block of 32, whose weights are row r of the matrix instruction
__device__ inline int matmul_feature(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

// 8 values of a row from k on, zeros from K on
template <typename T>
__device__ inline v4i matmul_load8(const T* row, int k, int K)
{
    if (k + 8 <= K) return *(const v4i_any*)(row + k);
    typedef short v8s __attribute__((ext_vector_type(8)));
    union {
        v4i v;
        v8s s;
    } x;
    x.v = v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < K) x.s[i] = ((const short*)row)[k + i];
    return x.v;
}

template <typename R>
__device__ inline void matmul_read(const R* p, int valid, float (&v)[16])
{
    if (valid >= 16) {
        typedef R any __attribute__((ext_vector_type(4), aligned(sizeof(R))));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const any x = ((const any*)p)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < valid ? (float)p[i] : 0.0f;
    }
}

template <typename O>
__device__ inline void matmul_write(O* p, int valid, const float (&v)[16])
{
    if (valid >= 16) {
        constexpr int N = 16 / sizeof(O);
        typedef O any __attribute__((ext_vector_type(N), aligned(sizeof(O))));
#pragma unroll
        for (int i = 0; i < 16 / N; ++i) {
            any x;
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = (O)v[N * i + j];
            ((any*)p)[i] = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < valid) p[i] = (O)v[i];
    }
}

// 16 neighbouring features from n0 on of row m
template <typename T>
__device__ inline void matmul_finish(const MatmulArgs& a, float (&v)[16], int m, int n0, void* out)
{
    const int valid = a.n - n0;
    if (m >= a.m || valid <= 0) return;
    if (a.bias) {
        float b[16];
        matmul_read(a.bias + n0, valid, b);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += b[i];
    }
    act_apply(v, a.act);
    if (a.residual) {
        float r[16];
        const int64_t at = m * a.r_pitch + n0;
        if (a.res_float) matmul_read((const float*)a.residual + at, valid, r);
        else matmul_read((const T*)a.residual + at, valid, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += r[i];
        act_apply(v, a.act2);
    }
    const int64_t at = m * a.o_pitch + n0;
    if (a.out_float) matmul_write((float*)out + at, valid, v);
    else matmul_write((T*)out + at, valid, v);
}

// 64 x 64 of the result to a workgroup, 32 x 32 to a wave, both operands straight from memory.
template <typename T>
__global__ __launch_bounds__(256) void matmul_direct_kernel(MatmulArgs a, const T* x, const T* w, void* out)
{
    typedef typename vec8<T>::type V;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m0 = blockIdx.y * 64 + (wave >> 1) * 32, n0 = blockIdx.x * 64 + (wave & 1) * 32;
    const int half = lane >> 5, r = lane & 31;
    const T* xr = x + (int64_t)min(m0 + r, a.m - 1) * a.a_pitch;
    const T* wr = w + (int64_t)min(n0 + matmul_feature(r), a.n - 1) * a.w_pitch;
    v16f acc = {};
#pragma unroll 4
    for (int k = 0; k < a.k; k += 16) {
        const v4i p = matmul_load8(wr, k + 8 * half, a.k), q = matmul_load8(xr, k + 8 * half, a.k);
        acc = mfma32(__builtin_bit_cast(V, p), __builtin_bit_cast(V, q), acc);
    }
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = acc[i];
    matmul_finish<T>(a, v, m0 + r, n0 + 16 * half, out);
}

MatmulPlan* matmul_plan(const cldnn_hip_engine_s& e, const cldnn_hip_matmul_desc& d, cldnn_hip_operator_info& info)
{
    const auto is_half = [](int dt) { return dt == CLDNN_HIP_F16 || dt == CLDNN_HIP_BF16; };
    CHIP_REQUIRE(d.m > 0 && d.n > 0 && d.k > 0, CLDNN_HIP_INVALID_ARG, "matmul: sizes must be positive");
    CHIP_REQUIRE(is_half(d.dtype), CLDNN_HIP_INVALID_ARG, "matmul: a and weights must be f16 or bf16");
    CHIP_REQUIRE(d.out_dtype == d.dtype || d.out_dtype == CLDNN_HIP_F32, CLDNN_HIP_INVALID_ARG, "matmul: the output must be of a's type or f32");
    CHIP_REQUIRE(d.residual_dtype == d.dtype || d.residual_dtype == CLDNN_HIP_F32 || d.residual_dtype == CLDNN_HIP_NO_TYPE, CLDNN_HIP_INVALID_ARG,
                 "matmul: the residual must be of a's type or f32");
    CHIP_REQUIRE(d.residual_dtype != CLDNN_HIP_NO_TYPE || d.residual_activation == CLDNN_HIP_ACT_NONE, CLDNN_HIP_INVALID_ARG,
                 "matmul: an activation of the sum without a residual");
    std::unique_ptr<MatmulPlan> plan(new MatmulPlan{});
    MatmulArgs& a = plan->a;
    a.m = d.m, a.n = d.n, a.k = d.k;
    const auto pitch = [](int64_t stride, int64_t dense) {
        CHIP_REQUIRE(stride == 0 || stride >= dense, CLDNN_HIP_INVALID_ARG, "matmul: a stride shorter than its row");
        return stride ? stride : dense;
    };
    a.a_pitch = pitch(d.a_stride, d.k), a.w_pitch = pitch(d.weights_stride, d.k);
    a.o_pitch = pitch(d.out_stride, d.n), a.r_pitch = pitch(d.residual_stride, d.n);
    a.act = make_act(d.activation, d.activation_m, d.activation_n, "matmul");
    a.act2 = make_act(d.residual_activation, d.residual_activation_m, d.residual_activation_n, "matmul");
    a.res_float = d.residual_dtype == CLDNN_HIP_F32, a.out_float = d.out_dtype == CLDNN_HIP_F32;
    // marks what the object has; enqueue puts the pointers there
    a.bias = d.has_bias ? (const float*)1 : nullptr, a.residual = d.residual_dtype != CLDNN_HIP_NO_TYPE ? (const void*)1 : nullptr;
    plan->dt = d.dtype;
    const int64_t out_size = a.out_float ? 4 : 2, res_size = !a.residual ? 0 : a.res_float ? 4 : 2;
    CHIP_REQUIRE((d.m + 63) / 64 <= 65535, CLDNN_HIP_UNSUPPORTED_SIZE, "matmul: too many rows");
    info.launches = 1, info.block = 256;
    info.grid = (int)((int64_t)((d.n + 63) / 64) * ((d.m + 63) / 64));
    info.ops = 2ll * d.m * d.n * d.k;
    info.bytes = 2 * ((int64_t)d.m * d.k + (int64_t)d.n * d.k) + (d.has_bias ? 4ll * d.n : 0) + (int64_t)d.m * d.n * (out_size + res_size);
    snprintf(info.kernel_name, sizeof info.kernel_name, "matmul_direct<64x64>");
    return plan.release();
}

void matmul_launch(hipStream_t s, const MatmulPlan& p, void* workspace, const void* x, const void* w, const float* bias, const void* residual, void* out)
{
    MatmulArgs a = p.a;
    CHIP_REQUIRE((!a.bias || bias) && (!a.residual || residual), CLDNN_HIP_INVALID_ARG, "null device pointer");
    check_aligned(x, 2, "a"), check_aligned(w, 2, "weights"), check_aligned(out, a.out_float ? 4 : 2, "output");
    if (a.bias) check_aligned(bias, 4, "bias"), a.bias = bias;
    if (a.residual) check_aligned(residual, a.res_float ? 4 : 2, "residual"), a.residual = residual;
    with_half(p.dt, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((matmul_direct_kernel<T>), dim3((a.n + 63) / 64, (a.m + 63) / 64), dim3(256), 0, s, a, (const T*)x, (const T*)w, out);
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(MatmulPlan* p) { delete p; }

}  // namespace chip
