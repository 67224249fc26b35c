// What the float operators share: data types, activations, the operator object.
#pragma once
#include <algorithm>
#include <cstdio>
#include <memory>
#include <string>
#include <type_traits>
#include <vector>

#include "../../include/cldnn_hip_ops.h"
#include "runtime.h"

namespace chip {

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float v4f;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float v16f;
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int v4i;
typedef __attribute__((__vector_size__(2 * sizeof(int)))) int v2i;
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
// the same 16 bytes at any address: the memory unit takes them unaligned
typedef v4i v4i_any __attribute__((aligned(2)));
typedef v2i v2i_any __attribute__((aligned(2)));

template <typename T> struct vec8;
template <> struct vec8<_Float16> { typedef v8h type; };
template <> struct vec8<__bf16> { typedef v8b type; };

__device__ inline v16f mfma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline v16f mfma32(v8b a, v8b b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline v4f mfma16(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline v4f mfma16(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// ----------------------------------------------------------------------------- loads into LDS
// buffer descriptor: base, no stride, 2 GiB - 1 bytes
__device__ inline v4i buffer_of(const void* p)
{
    const uint64_t at = (uint64_t)p;
    return v4i{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff), 0x7fffffff, 0x00020000};
}

__device__ inline uint32_t lds_address(const v4i* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) v4i*)p; }

// Lane t's 16 bytes at `offset` + `step` go to LDS at place t from `to` on.  Written out because the compiler, where it issues this
// load itself, waits for all loads under way in front of one of three LDS reads of a loop (1498 against 1090 us for 8192 x 8192 x
// 8192).  It has no result in registers; a wait for vmcnt, written out as well, is what it needs before anybody reads.
// The load takes its place from M0, and a scalar write of M0 needs a wait state in front of it, which the compiler leaves for its own
// loads and does not look for in here.
// M0 has no other user in these kernels: this device's LDS instructions do not read it, and no register is indexed.
__device__ inline void load_lds(v4i from, uint32_t to, int offset, int step)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(offset), "s"(from), "s"(step) : "memory");
}

// ----------------------------------------------------------------------------- activations
struct Act {
    int32_t kind;
    float m, n;
};

// v P(Z <= v) = max(v, 0) - |v| P(Z > |v|), without a difference of near equals on either side.  P(Z > a) = erfc(a / sqrt 2) / 2 by
// Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26 (error 1.5e-7), with the factors of 2 in its constants.
__device__ inline float act_gelu(float v)
{
    const float a = __builtin_fminf(__builtin_fabsf(v), 1e18f);  // infinity times no probability is no value
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, a, 1.0f));
    float p = __builtin_fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    p = __builtin_fmaf(p, t, 0.5f * 1.421413741f);
    p = __builtin_fmaf(p, t, 0.5f * -0.284496736f);
    p = __builtin_fmaf(p, t, 0.5f * 0.254829592f);
    const float u = 0.84932180f * v;  // sqrt(log2(e) / 2)
    const float q = p * t * __builtin_amdgcn_exp2f(-(u * u));
    return __builtin_fmaf(-a, q, v < 0.0f ? 0.0f : v);
}

template <int KIND>
__device__ inline float act_one(float v, float m, float n)
{
    if constexpr (KIND == CLDNN_HIP_ACT_RELU) return v < 0.0f ? 0.0f : v;  // NaN stays
    if constexpr (KIND == CLDNN_HIP_ACT_RELU_SLOPE) return v < 0.0f ? v * m : v;
    if constexpr (KIND == CLDNN_HIP_ACT_CLAMP) return v < m ? m : v > n ? n : v;
    if constexpr (KIND == CLDNN_HIP_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
    if constexpr (KIND == CLDNN_HIP_ACT_GELU) return act_gelu(v);
    if constexpr (KIND == CLDNN_HIP_ACT_GELU_TANH) {
        // (1 + tanh u) / 2 = 1 / (1 + exp(-2u)),  u = 0.79788456 (v + 0.044715 v^3)
        const float u = v * __builtin_fmaf(0.044715f * v, v, 1.0f);
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.30220818f * u));
    }
    return v;
}

// f(the activation as a constant): one uniform branch around whatever f does with it
template <typename F>
__device__ __forceinline__ void act_choose(int kind, F&& f)
{
    switch (kind) {
    case CLDNN_HIP_ACT_RELU: return f(std::integral_constant<int, CLDNN_HIP_ACT_RELU>());
    case CLDNN_HIP_ACT_RELU_SLOPE: return f(std::integral_constant<int, CLDNN_HIP_ACT_RELU_SLOPE>());
    case CLDNN_HIP_ACT_CLAMP: return f(std::integral_constant<int, CLDNN_HIP_ACT_CLAMP>());
    case CLDNN_HIP_ACT_SILU: return f(std::integral_constant<int, CLDNN_HIP_ACT_SILU>());
    case CLDNN_HIP_ACT_GELU: return f(std::integral_constant<int, CLDNN_HIP_ACT_GELU>());
    case CLDNN_HIP_ACT_GELU_TANH: return f(std::integral_constant<int, CLDNN_HIP_ACT_GELU_TANH>());
    default: return f(std::integral_constant<int, CLDNN_HIP_ACT_NONE>());
    }
}

// N values with one activation
template <int N>
__device__ inline void act_apply(float (&v)[N], const Act& a)
{
    act_choose(a.kind, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = act_one<decltype(kind)::value>(v[i], a.m, a.n);
    });
}

// ----------------------------------------------------------------------------- operator objects
enum OperatorKind { OP_GROUP_NORM, OP_MATMUL, OP_ROTARY, OP_ATTENTION };

struct NormPlan;
struct MatmulPlan;
struct RotaryPlan;
struct AttentionPlan;

}  // namespace chip

struct cldnn_hip_operator_s {
    std::atomic<int> refs{1};
    cldnn_hip_engine engine = nullptr;
    chip::OperatorKind kind{};
    void* workspace = nullptr;  // device memory
    cldnn_hip_operator_info info{};
    // what create worked out, one of them
    chip::NormPlan* norm = nullptr;
    chip::MatmulPlan* matmul = nullptr;
    chip::RotaryPlan* rotary = nullptr;
    chip::AttentionPlan* attention = nullptr;
    ~cldnn_hip_operator_s();
};

namespace chip {

// bytes of an element of the operators' float types; refuses others
inline int float_size(int dt, const char* what)
{
    switch (dt) {
    case CLDNN_HIP_F32: return 4;
    case CLDNN_HIP_F16:
    case CLDNN_HIP_BF16: return 2;
    default: throw error(CLDNN_HIP_INVALID_ARG, std::string(what) + ": data must be f32, f16 or bf16");
    }
}

// f(T()) for the element type of `dt`
template <typename F>
void with_half(int dt, F&& f)
{
    if (dt == CLDNN_HIP_F16) f(_Float16());
    else f(__bf16());
}
template <typename F>
void with_float(int dt, F&& f)
{
    if (dt == CLDNN_HIP_F32) f(float());
    else with_half(dt, f);
}

// Each plan: what create works out from a description (refusing what is wrong), and the launch.
NormPlan* norm_plan(const cldnn_hip_engine_s& e, const cldnn_hip_group_norm_desc& d, cldnn_hip_operator_info& info);
void norm_launch(hipStream_t s, const NormPlan& p, void* workspace, const void* in, const float* scale, const float* shift, void* out);
MatmulPlan* matmul_plan(const cldnn_hip_engine_s& e, const cldnn_hip_matmul_desc& d, cldnn_hip_operator_info& info);
void matmul_launch(hipStream_t s, const MatmulPlan& p, void* workspace, const void* a, const void* w, const float* bias, const void* residual, void* out);
// init: what the object's workspace starts with
RotaryPlan* rotary_plan(const cldnn_hip_engine_s& e, const cldnn_hip_rotary_desc& d, cldnn_hip_operator_info& info, std::vector<char>& init);
void rotary_launch(hipStream_t s, const RotaryPlan& p, const void* workspace, const void* q, const void* k, const void* positions, void* q_out, void* k_out);
AttentionPlan* attention_plan(const cldnn_hip_engine_s& e, const cldnn_hip_attention_desc& d, cldnn_hip_operator_info& info);
void attention_launch(hipStream_t s, const AttentionPlan& p, void* workspace, const void* q, const void* k, const void* v, const int32_t* lengths,
                      const void* bias, void* out);
void free_plan(NormPlan*);
void free_plan(MatmulPlan*);
void free_plan(RotaryPlan*);
void free_plan(AttentionPlan*);

inline void check_aligned(const void* p, size_t to, const char* what)
{
    CHIP_REQUIRE(((uintptr_t)p & (to - 1)) == 0, CLDNN_HIP_INVALID_ARG, std::string(what) + " is not aligned to " + std::to_string(to) + " bytes");
}

// the runtime counts a grid's threads along an axis in 32 bits
inline void check_grid(int64_t blocks, int threads, const char* what)
{
    CHIP_REQUIRE(blocks < (1ll << 32) / threads, CLDNN_HIP_UNSUPPORTED_SIZE, std::string(what) + ": too large");
}

inline Act make_act(int32_t kind, float m, float n, const char* what)
{
    CHIP_REQUIRE(kind >= CLDNN_HIP_ACT_NONE && kind <= CLDNN_HIP_ACT_GELU_TANH, CLDNN_HIP_INVALID_ARG, std::string(what) + ": unknown activation");
    CHIP_REQUIRE(kind != CLDNN_HIP_ACT_CLAMP || m <= n, CLDNN_HIP_INVALID_ARG, std::string(what) + ": clamp with its bounds the wrong way round");
    return Act{kind, m, n};
}

}  // namespace chip
