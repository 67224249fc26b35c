// Rows held in registers: a row belongs to a group of LANES threads, lane l of which has the vectors l, l + LANES, .. of 8 values.  The
// last vector of a row that is no whole vectors lies over the one before it, so that all loads are whole; the values that it shares
// are the other lane's (RowVector::from).  (One element at a time, the last vectors of 25088 x 1100 doubled the time of a norm.)
// What the operators that go over rows share: loads and stores of any float type at any element's address, sums and maxima over a row,
// quantised rows.
#pragma once
#include "ops_s8.h"

namespace chip {

// Values of the longest row: 512 threads leave 256 registers to each, which 8 vectors of two tensors of f32 and the values made of them fit
// (1024 threads with 4 vectors each, in 128 registers, keep some in scratch memory).
constexpr int ROW_MOST = 8 * 512 * 8;
constexpr int64_t ROW_PAST = 32 << 20;  // bytes that the dies' caches hold together

// Waves of a SIMD that a kernel with NV vectors a lane leaves registers for: what covers a row's trips to memory is other rows.
constexpr int row_waves(int NV) { return NV == 1 ? 7 : NV == 2 ? 6 : NV == 3 ? 4 : NV == 4 ? 3 : 2; }

// The vector of a lane: values c .. c + 7 of the row, of which those from `from` on, and below C, are the lane's.
struct RowVector {
    int c, from;
    __device__ __forceinline__ bool whole(int C) const { return from == 0 && C >= 8; }
    __device__ __forceinline__ bool has(int i, int C) const { return i >= from && c + i < C; }
};

// f(i, vector) for the vectors of a lane.  The first SURE of them are whole for every lane.  One behind the row is the row's last
// vector, with nothing in it that is the lane's: the program has no branch around what is done with it.
template <int LANES, int NV, int SURE, typename F>
__device__ __forceinline__ void row_each(int lane, int C, F&& f)
{
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * LANES) * 8, at = i < SURE ? c : min(c, max(C - 8, 0));
        f(i, RowVector{at, c - at});
    }
}

// the length of a row, of which the compiler may know that longer shapes have at least a vector
template <int LANES, int SURE>
__device__ __forceinline__ int row_length(int C)
{
    if constexpr (LANES > 16 || SURE > 0) __builtin_assume(C > 128);
    return C;
}

// what is not the lane's becomes zero
__device__ __forceinline__ void row_mask(const RowVector& of, int C, float (&v)[8])
{
    if (!of.whole(C))
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = of.has(i, C) ? v[i] : 0.0f;
}

// 8 values as they lie in memory: f32 takes both, the 16-bit types the first.  WIDE: it may be f32.
template <bool WIDE>
struct RowRaw {
    v4i a, b;
};
template <>
struct RowRaw<false> {
    v4i a;
};

// The values c .. c + 7 of a row, which is shorter than that if it has less than 8: zeros then.
template <bool WIDE>
__device__ __forceinline__ RowRaw<WIDE> row_load(const void* row, int type, int c, int C)
{
    typedef v4i any4 __attribute__((aligned(4)));
    RowRaw<WIDE> x;
    if constexpr (WIDE)
        if (type == CLDNN_HIP_F32) {
            const float* p = (const float*)row + c;
            if (C >= 8) x.a = ((const any4*)p)[0], x.b = ((const any4*)p)[1];
            else {
                x.a = x.b = v4i{0, 0, 0, 0};
                for (int i = 0; i < C; ++i) (i < 4 ? x.a : x.b)[i & 3] = __builtin_bit_cast(int, p[i]);
            }
            return x;
        }
    const uint16_t* p = (const uint16_t*)row + c;
    if (C >= 8) x.a = *(const v4i_any*)p;
    else {
        x.a = v4i{0, 0, 0, 0};
        for (int i = 0; i < C; ++i) x.a[i / 2] |= (int)p[i] << (16 * (i & 1));
    }
    return x;
}

template <bool WIDE>
__device__ __forceinline__ void row_values(const RowRaw<WIDE>& x, int type, float (&v)[8])
{
    if constexpr (WIDE)
        if (type == CLDNN_HIP_F32) {
            const v4f a = __builtin_bit_cast(v4f, x.a), b = __builtin_bit_cast(v4f, x.b);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
            return;
        }
    if (type == CLDNN_HIP_F16) {
        const v8h h = __builtin_bit_cast(v8h, x.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
        const v8b h = __builtin_bit_cast(v8b, x.a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    }
}

__device__ __forceinline__ void row_floats(const float* row, int c, int C, float (&v)[8]) { row_values(row_load<true>(row, CLDNN_HIP_F32, c, C), CLDNN_HIP_F32, v); }

// PAST: past the caches
template <bool PAST, typename V, typename A>
__device__ __forceinline__ void row_write(A* p, const V& x)
{
    if constexpr (PAST) __builtin_nontemporal_store((A)x, p);
    else *p = x;
}

template <bool PAST, typename T>
__device__ __forceinline__ void row_store_as(T* row, const RowVector& of, int C, const float (&v)[8])
{
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    constexpr int W = 16 / sizeof(T);
    T* p = row + of.c;
    if (of.whole(C)) {
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            vec x;
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] = (T)v[W * j + i];
            row_write<PAST>((any*)p + j, x);
        }
    } else if (of.from < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (of.has(i, C)) p[i] = (T)v[i];
    }
}

// rounded once, to the type
template <bool PAST>
__device__ __forceinline__ void row_store(void* row, int type, const RowVector& of, int C, const float (&v)[8])
{
    if (type == CLDNN_HIP_F32) row_store_as<PAST>((float*)row, of, C, v);
    else if (type == CLDNN_HIP_F16) row_store_as<PAST>((_Float16*)row, of, C, v);
    else row_store_as<PAST>((__bf16*)row, of, C, v);
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

// the largest magnitude; NaN where a value is NaN
template <int LANES>
__device__ __forceinline__ float row_most(float v, float* slot)
{
    return row_all<LANES>(v, slot, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
}

__device__ __forceinline__ float row_magnitude(const float (&v)[8], float most)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __builtin_elementwise_maximum(most, __builtin_fabsf(v[i]));
    return most;
}

// ----------------------------------------------------------------------------- quantised rows
struct RowSteps {
    float inverse, scale;
    bool bad;  // a value that is not finite
};

__device__ __forceinline__ RowSteps row_steps(float most)
{
    RowSteps s{0.0f, 0.0f, !(most < __builtin_inff())};
    if (s.bad) s.scale = __builtin_nanf("");
    else if (most >= 0x1p-120f) s.inverse = 127.0f / most, s.scale = most / 127.0f;  // 127 * 2^120 is finite
    return s;
}

// Rounds by adding 3 * 2^22: what is left in the low byte is the whole number in two's complement.  |v * inverse| is 127 and a rounding
// at most.
__device__ __forceinline__ void row_store_s8(int8_t* row, const RowVector& of, int C, const float (&v)[8], const RowSteps& s)
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
    int8_t* p = row + of.c;
    if (of.whole(C)) *(any*)p = q;
    else if (of.from < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (of.has(i, C)) p[i] = (int8_t)((uint32_t)q[i / 4] >> (8 * (i & 3)));
    }
}

// ----------------------------------------------------------------------------- which group of threads takes a row
struct RowShape {
    int lanes, vectors;  // of a row; vectors a lane
    int threads() const { return std::max(lanes, 256); }
    int rows() const { return threads() / lanes; }  // of a workgroup
    int64_t blocks(int64_t all) const { return (all + rows() - 1) / rows(); }
};

// f(lanes, vectors, SURE as constants) if that shape holds a row of C values.  An operator tries its shapes in order; SURE is what the one
// before leaves for sure.
template <int LANES, int NV, int SURE, typename F>
bool try_row_shape(int C, F&& f)
{
    if ((C + 7) / 8 > LANES * NV) return false;
    f(std::integral_constant<int, LANES>(), std::integral_constant<int, NV>(), std::integral_constant<int, SURE>());
    return true;
}

}  // namespace chip
