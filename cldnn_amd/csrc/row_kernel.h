// Rows held in registers: a row belongs to a group of LANES threads, lane l of which has the vectors l, l + LANES, .. of 8 values.
// What the operators that go over rows share: loads and stores of any float type at any element's address, sums and maxima over a row,
// quantised rows.
#pragma once
#include "ops_s8.h"

namespace chip {

// Values of the longest row: 512 threads leave 256 registers to each, which 8 vectors of two tensors of f32 and the values made of them fit
// (1024 threads with 4 vectors each, in 128 registers, keep some in scratch memory).
constexpr int ROW_MOST = 8 * 512 * 8;

// 8 values as they lie in memory: f32 takes both, the 16-bit types the first
struct RowRaw {
    v4i a, b;
};

// The values c .. c + 7 of a row; zeros from C on.
__device__ __forceinline__ RowRaw row_load(const void* row, int type, int c, int C)
{
    typedef v4i any4 __attribute__((aligned(4)));
    RowRaw x;
    if (type == CLDNN_HIP_F32) {
        const float* p = (const float*)row + c;
        if (c + 8 <= C) x.a = ((const any4*)p)[0], x.b = ((const any4*)p)[1];
        else {
            x.a = x.b = v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (c + i < C) x.a[i] = __builtin_bit_cast(int, p[i]);
                if (c + 4 + i < C) x.b[i] = __builtin_bit_cast(int, p[4 + i]);
            }
        }
    } else {
        const uint16_t* p = (const uint16_t*)row + c;
        if (c + 8 <= C) x.a = *(const v4i_any*)p;
        else {
            x.a = v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < C) x.a[i / 2] |= (int)p[i] << (16 * (i & 1));
        }
    }
    return x;
}

__device__ __forceinline__ void row_values(const RowRaw& x, int type, float (&v)[8])
{
    if (type == CLDNN_HIP_F32) {
        const v4f a = __builtin_bit_cast(v4f, x.a), b = __builtin_bit_cast(v4f, x.b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else if (type == CLDNN_HIP_F16) {
        const v8h h = __builtin_bit_cast(v8h, x.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
        const v8b h = __builtin_bit_cast(v8b, x.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    }
}

__device__ __forceinline__ void row_floats(const float* row, int c, int C, float (&v)[8]) { row_values(row_load(row, CLDNN_HIP_F32, c, C), CLDNN_HIP_F32, v); }

template <typename T>
__device__ __forceinline__ void row_store_as(T* p, int valid, const float (&v)[8])
{
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    constexpr int W = 16 / sizeof(T);
    if (valid >= 8) {
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            vec x;
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] = (T)v[W * j + i];
            ((any*)p)[j] = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}

// rounded once, to the type
__device__ __forceinline__ void row_store(void* row, int type, int c, int C, const float (&v)[8])
{
    if (type == CLDNN_HIP_F32) row_store_as((float*)row + c, C - c, v);
    else if (type == CLDNN_HIP_F16) row_store_as((_Float16*)row + c, C - c, v);
    else row_store_as((__bf16*)row + c, C - c, v);
}

// ----------------------------------------------------------------------------- over a row
// op over all lanes of the row's group, which call this together; `slot` of LDS is used once.  A fixed order: the same bits every time.
template <int LANES, typename T, typename F>
__device__ __forceinline__ T row_all(T v, T* slot, F&& op)
{
    const auto dpp = [&](auto ctrl) { return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true)); };
    v = op(v, dpp(std::integral_constant<int, 0xb1>()));   // lanes 1 apart
    v = op(v, dpp(std::integral_constant<int, 0x4e>()));   // 2 apart
    v = op(v, dpp(std::integral_constant<int, 0x141>()));  // the other four of eight
    v = op(v, dpp(std::integral_constant<int, 0x140>()));  // the other eight of sixteen
    if constexpr (LANES > 16) {
        v = op(v, __shfl_xor(v, 16));
        v = op(v, __shfl_xor(v, 32));
    }
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = op(v, slot[i]);
    }
    return v;
}

template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slot)
{
    return row_all<LANES>(v, slot, [](float a, float b) { return a + b; });
}

// magnitudes as the bits of a float, which compare like whole numbers: NaN is above infinity
template <int LANES>
__device__ __forceinline__ uint32_t row_most(uint32_t v, float* slot)
{
    return row_all<LANES>(v, (uint32_t*)slot, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint32_t row_magnitude(const float (&v)[8], uint32_t most)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t m = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
        most = m > most ? m : most;
    }
    return most;
}

// ----------------------------------------------------------------------------- quantised rows
struct RowSteps {
    float inverse, scale;
    bool bad;  // a value that is not finite
};

__device__ __forceinline__ RowSteps row_steps(uint32_t most_bits)
{
    const float most = __builtin_bit_cast(float, most_bits);
    RowSteps s{0.0f, 0.0f, most_bits >= 0x7f800000u};
    if (s.bad) s.scale = __builtin_nanf("");
    else if (most >= 0x1p-120f) s.inverse = 127.0f / most, s.scale = most / 127.0f;  // 127 * 2^120 is finite
    return s;
}

// Rounds by adding 3 * 2^22: what is left in the low byte is the whole number in two's complement.  |v * inverse| is 127 and a rounding
// at most.
__device__ __forceinline__ void row_store_s8(int8_t* p, int valid, const float (&v)[8], const RowSteps& s)
{
#pragma clang fp contract(off)
    uint32_t bits[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = v[i] * s.inverse;
        bits[i] = __builtin_bit_cast(uint32_t, x + 12582912.0f);
    }
    v2i q;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t lo = __builtin_amdgcn_perm(bits[4 * j + 1], bits[4 * j], 0x0c0c0400), hi = __builtin_amdgcn_perm(bits[4 * j + 3], bits[4 * j + 2], 0x0c0c0400);
        q[j] = s.bad ? 0 : (int)(lo | hi << 16);
    }
    typedef v2i any __attribute__((aligned(1)));
    if (valid >= 8) *(any*)p = q;
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = (int8_t)((uint32_t)q[i / 4] >> (8 * (i & 3)));
    }
}

// ----------------------------------------------------------------------------- which group of threads takes a row
struct RowShape {
    int lanes, vectors;  // of a row; vectors a lane
    int threads() const { return std::max(lanes, 256); }
    int rows() const { return threads() / lanes; }  // of a workgroup
    int64_t blocks(int64_t all) const { return (all + rows() - 1) / rows(); }
};

// rows of C values, at most ROW_MOST
inline RowShape row_shape(int C)
{
    const int vectors = (C + 7) / 8;
    for (const RowShape s : {RowShape{16, 1}, RowShape{64, 1}, RowShape{64, 2}, RowShape{64, 4}, RowShape{256, 2}, RowShape{256, 4}, RowShape{512, 4}})
        if (vectors <= s.lanes * s.vectors) return s;
    return RowShape{512, 8};
}

// f(lanes, vectors as constants)
template <typename F>
void with_row_shape(const RowShape& s, F&& f)
{
    const auto c = [&](auto lanes, auto vectors) { f(lanes, vectors); };
    typedef std::integral_constant<int, 16> L16;
    typedef std::integral_constant<int, 64> L64;
    typedef std::integral_constant<int, 256> L256;
    typedef std::integral_constant<int, 512> L512;
    typedef std::integral_constant<int, 1> V1;
    typedef std::integral_constant<int, 2> V2;
    typedef std::integral_constant<int, 4> V4;
    typedef std::integral_constant<int, 8> V8;
    switch (s.lanes * 8 + s.vectors) {
    case 16 * 8 + 1: return c(L16(), V1());
    case 64 * 8 + 1: return c(L64(), V1());
    case 64 * 8 + 2: return c(L64(), V2());
    case 64 * 8 + 4: return c(L64(), V4());
    case 256 * 8 + 2: return c(L256(), V2());
    case 256 * 8 + 4: return c(L256(), V4());
    case 512 * 8 + 4: return c(L512(), V4());
    default: return c(L512(), V8());
    }
}

}  // namespace chip
