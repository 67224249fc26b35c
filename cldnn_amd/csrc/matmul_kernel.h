// The kernels of the matrix products, for operands of f16, bf16 and int8: out = act2(act(a w^T + bias) + residual).
//
// The weights are the row operand of the matrix instruction, so that a lane ends with neighbouring features of one row of the
// result: whole 16-byte stores, and a bias and a residual that are read the same way.
#pragma once
#include "ops_common.h"

namespace chip {

struct MatmulArgs {
    int32_t m, n, k;
    int64_t a_pitch, w_pitch, o_pitch, r_pitch;
    const float* bias;
    const void* residual;  // nullptr: none
    Act act, act2;
    int32_t tiles, tiles_m, tiles_n;  // of the result
    int32_t band;                     // rows of tiles in a band
    int32_t splits;                   // workgroups that split K for each tile: their sums go to part[split][m][n]
    void* part;                       // of the operands' sums: float or int32_t
};

// ... of the product of float operands: result and residual are of their type or f32
struct MatmulFloatArgs : MatmulArgs {
    int32_t res_float, out_float;
};

// ... and of int8 operands: scales of the rows of a and of the weights' rows, out types apart from the operands'
struct MatmulS8Args : MatmulArgs {
    const float *a_scales, *w_scales;  // nullptr: 1
    int32_t a_each, w_each;            // 1: one to a row; 0: one for all
    int32_t out_type, res_type;        // CLDNN_HIP_F32, F16, BF16
    int32_t out_runs;                  // result and residual are whole runs of matmul_run values at any place of a tile
    int32_t past;                      // the result of a large product goes past the caches
};

// What the kernels ask of an operand's type: a 16-byte piece as the matrix instruction takes it, its sums, the arguments of its product.
// An int8 piece holds twice the values, and the instruction multiplies twice as many in the same time: both types go through the same
// bytes in the same order.
template <typename T> struct MatmulType {
    typedef typename vec8<T>::type V;
    typedef v4i_any Any;  // a piece at any element's address
    typedef v4f Sum;
    typedef float One;
    typedef MatmulFloatArgs Args;
    static constexpr int E = 8;  // values of a piece
    static constexpr bool SHORT = false;  // form of the activations
};
template <> struct MatmulType<int8_t> {
    typedef v4i V;
    typedef v4i Any __attribute__((aligned(1)));
    typedef v4i Sum;
    typedef int32_t One;
    typedef MatmulS8Args Args;
    static constexpr int E = 16;
    static constexpr bool SHORT = true;
};
__device__ inline v4i mfma16(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

constexpr int MATMUL_PACK_THREADS = 256;

// a piece of a row from k on, zeros from K on
template <typename T>
__device__ inline v4i matmul_load(const T* row, int k, int K)
{
    constexpr int E = MatmulType<T>::E;
    typedef typename MatmulType<T>::Any any;
    if (k + E <= K) return *(const any*)(row + k);
    if constexpr (E == 16)
        if (K >= E) {  // the row's last piece, moved (one value at a time: 13.7 us instead of 6.8 for 1000 x 127 -> 1000)
            const unsigned __int128 last = __builtin_bit_cast(unsigned __int128, (v4i)*(const any*)(row + K - E));
            return __builtin_bit_cast(v4i, k < K ? last >> (8 * (k + E - K)) : (unsigned __int128)0);
        }
    typedef std::conditional_t<E == 8, short, signed char> I;
    typedef I vE __attribute__((ext_vector_type(E)));
    union {
        v4i v;
        vE s;
    } x;
    x.v = v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (k + i < K) x.s[i] = ((const I*)row)[k + i];
    return x.v;
}

template <typename R, typename V, int N>
__device__ __forceinline__ void matmul_read(const R* p, int valid, V (&v)[N])
{
    if (valid >= N) {
        constexpr int W = 16 / sizeof(R) < N ? 16 / sizeof(R) : N;
        typedef R any __attribute__((ext_vector_type(W), aligned(sizeof(R))));
#pragma unroll
        for (int i = 0; i < N / W; ++i) {
            const any x = ((const any*)p)[i];
#pragma unroll
            for (int j = 0; j < W; ++j) v[W * i + j] = (V)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? (V)p[i] : (V)0;
    }
}

template <typename O, typename V, int N>
__device__ __forceinline__ void matmul_write(O* p, int valid, const V (&v)[N])
{
    if (valid >= N) {
        constexpr int W = 16 / sizeof(O) < N ? 16 / sizeof(O) : N;
        typedef O any __attribute__((ext_vector_type(W), aligned(sizeof(O))));
#pragma unroll
        for (int i = 0; i < N / W; ++i) {
            any x;
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = (O)v[W * i + j];
            ((any*)p)[i] = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = (O)v[i];
    }
}

// N neighbouring features from n0 on of row m behind their activation: the residual, the result
template <typename T, int N>
__device__ __forceinline__ void matmul_write_row(const MatmulFloatArgs& a, float (&v)[N], int m, int n0, void* out)
{
    const int valid = a.n - n0;
    if (m >= a.m || valid <= 0) return;
    if (a.residual) {
        float r[N];
        const int64_t at = m * a.r_pitch + n0;
        if (a.res_float) matmul_read((const float*)a.residual + at, valid, r);
        else matmul_read((const T*)a.residual + at, valid, r);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += r[i];
        act_apply(v, a.act2);
    }
    const int64_t at = m * a.o_pitch + n0;
    if (a.out_float) matmul_write((float*)out + at, valid, v);
    else matmul_write((T*)out + at, valid, v);
}

// The same for int8 operands, where the types of result and residual are free of theirs.
template <typename T, int N>
__device__ __forceinline__ void matmul_write_row(const MatmulS8Args& a, float (&v)[N], int m, int n0, void* out)
{
    const int valid = a.n - n0;
    if (m >= a.m || valid <= 0) return;
    if (a.residual) {
        float r[N];
        const int64_t at = m * a.r_pitch + n0;
        if (a.res_type == CLDNN_HIP_F32) matmul_read((const float*)a.residual + at, valid, r);
        else if (a.res_type == CLDNN_HIP_F16) matmul_read((const _Float16*)a.residual + at, valid, r);
        else matmul_read((const __bf16*)a.residual + at, valid, r);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += r[i];
        act_apply<MatmulType<T>::SHORT>(v, a.act2);
    }
    const int64_t at = m * a.o_pitch + n0;
    if (a.out_type == CLDNN_HIP_F32) matmul_write((float*)out + at, valid, v);
    else if (a.out_type == CLDNN_HIP_F16) matmul_write((_Float16*)out + at, valid, v);
    else matmul_write((__bf16*)out + at, valid, v);
}

// What the sums of N neighbouring features from n on become: themselves,
template <typename T, int N>
struct MatmulColumns {
    __device__ __forceinline__ MatmulColumns(const MatmulArgs&, int) {}
    __device__ __forceinline__ float value(int, float sum, float) const { return sum; }
};
// ... or, of int8 operands, times the scales of row and feature.  The sum of whole numbers is exact, and rounded once where it does not
// fit 24 bits; each factor rounds once.
template <int N>
struct MatmulColumns<int8_t, N> {
    float scale[N];
    __device__ __forceinline__ MatmulColumns(const MatmulS8Args& a, int n)
    {
        const float all = a.w_scales && !a.w_each ? *a.w_scales : 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) scale[i] = all;
        if (a.w_each && n < a.n) matmul_read(a.w_scales + n, a.n - n, scale);
    }
    __device__ __forceinline__ float value(int i, int32_t sum, float row) const { return (float)sum * row * scale[i]; }
};
__device__ __forceinline__ float matmul_row_scale(const MatmulArgs&, int) { return 1.0f; }
__device__ __forceinline__ float matmul_row_scale(const MatmulS8Args& a, int m) { return a.a_scales ? a.a_scales[a.a_each ? min(m, a.m - 1) : 0] : 1.0f; }

// Tiles are dealt to the accelerator dies in turn (workgroup i runs on die i % 8): each die gets a run of neighbouring tiles.  A
// run goes through bands of a.band rows of tiles, down each column of a band, so that the tiles that a die works on at a time are
// a block whose operands its own L2 serves: 32 tiles in a row read 33 tiles' operands, 4 x 8 read 12.
__device__ inline void matmul_place(const MatmulArgs& a, int i, int& tm, int& tn)
{
    const int die = i & 7, each = a.tiles >> 3, more = a.tiles & 7;
    const int tile = die * each + min(die, more) + (i >> 3);
    const int band = tile / (a.band * a.tiles_n), in = tile - band * a.band * a.tiles_n;
    const int rows = min(a.band, a.tiles_m - band * a.band);
    tn = in / rows;
    tm = band * a.band + in - tn * rows;
}

// all of this wave's loads have landed but the newest N, its LDS reads are done, and so for every wave
template <int N>
__device__ inline void matmul_arrive()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ inline void matmul_meet()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Few rows, or few tiles: 16 FT features x 16 PT rows to a workgroup, whose waves split K in runs of U steps of 32; both operands
// straight from memory into the registers that the matrix instruction reads; the partial sums meet in LDS.  Of a run of 16 steps the
// compiler keeps twelve loads, six steps, under way (70 registers) and lets them run out at its end.  Bound by the weights: 1 x 25088
// -> 4096 39 us, 5.3 TB/s, a large copy's rate; with 16 rows 55 us, their values being as many bytes again from the die's L2.  Of int8, steps
// of 64 and half the bytes: 21 and 29 us.
template <typename T, int FT, int PT, int U, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void matmul_split_kernel(typename MatmulType<T>::Args a, const T* x, const T* w, void* out)
{
    typedef MatmulType<T> Type;
    typedef typename Type::V V;
    typedef typename Type::Sum Sum;
    typedef typename Type::One One;
    typedef typename Type::Any any;
    constexpr int TILE = 256 * FT * PT, E = Type::E, STEP = 4 * E;
    __shared__ One sums[WAVES][TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    int tm, tn;
    matmul_place(a, blockIdx.x, tm, tn);
    const int m0 = tm * 16 * PT, n0 = tn * 16 * FT;
    const T *xr[PT], *wr[FT];
#pragma unroll
    for (int i = 0; i < PT; ++i) xr[i] = x + (int64_t)min(m0 + 16 * i + r, a.m - 1) * a.a_pitch + E * q;
#pragma unroll
    for (int i = 0; i < FT; ++i) wr[i] = w + (int64_t)min(n0 + 16 * i + r, a.n - 1) * a.w_pitch + E * q;
    Sum acc[FT][PT] = {};
    const int whole = a.k / (STEP * U);  // runs of U full steps, dealt to the waves in turn
    const int worker = blockIdx.y * WAVES + wave, workers = a.splits * WAVES;
    for (int run = worker; run < whole; run += workers) {
        const int k = run * STEP * U;
        v4i wf[U][FT], xf[U][PT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < FT; ++i) wf[u][i] = *(const any*)(wr[i] + k + STEP * u);
#pragma unroll
            for (int i = 0; i < PT; ++i) xf[u][i] = *(const any*)(xr[i] + k + STEP * u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int j = 0; j < PT; ++j) acc[i][j] = mfma16(__builtin_bit_cast(V, wf[u][i]), __builtin_bit_cast(V, xf[u][j]), acc[i][j]);
    }
    // the steps behind the runs, one to a wave
    const int steps = a.k / STEP + (a.k % STEP != 0);
    for (int step = whole * U + (worker - whole % workers + workers) % workers; step < steps; step += workers) {
        const int k = step * STEP;
        v4i wf[FT], xf[PT];
#pragma unroll
        for (int i = 0; i < FT; ++i) wf[i] = matmul_load(wr[i] - E * q, k + E * q, a.k);
#pragma unroll
        for (int i = 0; i < PT; ++i) xf[i] = matmul_load(xr[i] - E * q, k + E * q, a.k);
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int j = 0; j < PT; ++j) acc[i][j] = mfma16(__builtin_bit_cast(V, wf[i]), __builtin_bit_cast(V, xf[j]), acc[i][j]);
    }
    // [row][feature], so that a thread's N values are neighbouring features
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < PT; ++j) *(Sum*)&sums[wave][(16 * j + r) * 16 * FT + 16 * i + 4 * q] = acc[i][j];
    __syncthreads();
    constexpr int N = TILE / (64 * WAVES) < 1 ? 1 : TILE / (64 * WAVES) > 16 ? 16 : TILE / (64 * WAVES);
    static_assert(16 * FT % N == 0, "a thread's values lie in one row");
    for (int at = threadIdx.x * N; at < TILE; at += 64 * WAVES * N) {
        One sum[N];
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = sums[0][at + i];
#pragma unroll
        for (int s = 1; s < WAVES; ++s)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += sums[s][at + i];
        const int row = at / (16 * FT), n = n0 + at - row * 16 * FT;
        if (a.splits > 1) {
            if (m0 + row < a.m && n < a.n) matmul_write((One*)a.part + ((int64_t)blockIdx.y * a.m + m0 + row) * a.n + n, a.n - n, sum);
            continue;
        }
        float v[N];
        const MatmulColumns<T, N> columns(a, n);
        const float scale = matmul_row_scale(a, m0 + row);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = columns.value(i, sum[i], scale);
        if (a.bias && n < a.n) {
            float b[N];
            matmul_read(a.bias + n, a.n - n, b);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += b[i];
        }
        act_apply<MatmulType<T>::SHORT>(v, a.act);
        matmul_write_row<T>(a, v, m0 + row, n, out);
    }
}

// The sums of the workgroups that split K, joined in their order: four features of a row to a thread.
template <typename T>
__global__ __launch_bounds__(256) void matmul_join_kernel(typename MatmulType<T>::Args a, void* out)
{
    const int across = (a.n + 3) / 4, i = blockIdx.x * 256 + threadIdx.x, m = i / across, n = (i - m * across) * 4;
    if (m >= a.m) return;
    typedef typename MatmulType<T>::One One;
    const One* part = (const One*)a.part;
    One sum[4];
    matmul_read(part + (int64_t)m * a.n + n, a.n - n, sum);
#pragma unroll 4
    for (int s = 1; s < a.splits; ++s) {
        One x[4];
        matmul_read(part + ((int64_t)s * a.m + m) * a.n + n, a.n - n, x);
#pragma unroll
        for (int l = 0; l < 4; ++l) sum[l] += x[l];
    }
    float v[4];
    const MatmulColumns<T, 4> columns(a, n);
    const float scale = matmul_row_scale(a, m);
#pragma unroll
    for (int l = 0; l < 4; ++l) v[l] = columns.value(l, sum[l], scale);
    if (a.bias) {
        float b[4];
        matmul_read(a.bias + n, a.n - n, b);
#pragma unroll
        for (int l = 0; l < 4; ++l) v[l] += b[l];
    }
    act_apply<MatmulType<T>::SHORT>(v, a.act);
    matmul_write_row<T>(a, v, m, n, out);
}

// ----------------------------------------------------------------------------- the end of a tile of int8 operands
// Values of a run, of results of `size` bytes: 16 bytes, which a lane stores as one piece beside those of its neighbours.  Four lanes write
// 64 bytes without a gap then; 16 neighbours to a lane, as the float products have them, are written in pieces 32 bytes apart, and 25088 x
// 1024 -> 4096 took twice the requests to memory.
constexpr int matmul_run(int size) { return 16 / size; }

// Where the g-th four of a lane's 16 values lie among the wave's 64 features.
__device__ inline int matmul_four(const MatmulS8Args& a, int g, int q) { return a.out_type == CLDNN_HIP_F32 ? 16 * g + 4 * q : 32 * (g >> 1) + 8 * q + 4 * (g & 1); }
__device__ inline int matmul_feature(const MatmulS8Args& a, int b) { return matmul_four(a, b >> 4, b >> 2 & 3) + (b & 3); }

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// f(T()) for one of the float types
template <typename F>
__device__ __forceinline__ void matmul_typed(int type, F&& f)
{
    if (type == CLDNN_HIP_F32) f(float());
    else if (type == CLDNN_HIP_F16) f(_Float16());
    else f(__bf16());
}

// A lane's 16 values of a row of the residual as they lie in memory; 16-bit types fill half.
typedef uint32_t v16u __attribute__((ext_vector_type(16)));
template <typename T>
__device__ __forceinline__ void matmul_add_row(const v16u& row, float (&v)[16])
{
    typedef T vec __attribute__((ext_vector_type(64 / sizeof(T))));
    const vec x = __builtin_bit_cast(vec, row);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += (float)x[i];
}

// The sums of a wave, 16 MB rows from m on x 64 features from n on: scales, bias, activation, residual, its activation, the result.  The
// residual's row is asked for one row ahead.  A result that is no whole runs is written in fours at any element's address (through LDS, one
// element to a lane: 4888 x 192 -> 4471 in f16 with a gelu 51 us, 33 now, 889 x 240 -> 5587 in bf16 19.5 and 13.6).
template <int MB>
__device__ __forceinline__ void matmul_finish_s8(const MatmulS8Args& a, const v4i (&sum)[4][MB], int m, int n, int lane, void* out)
{
    const int q = lane >> 4, r = lane & 15;
    const bool fours = a.out_type == CLDNN_HIP_F32;
    const int res_size = a.res_type == CLDNN_HIP_F32 ? 4 : 2, out_size = fours ? 4 : 2;
    const auto buffer = [&](const void* base, int64_t pitch, int size) {
        return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(base) + (m * pitch + n) * size, 0, 0x7fffffff, 0x00020000);
    };
    const auto from = buffer(a.residual, a.r_pitch, res_size), to = buffer(out, a.o_pitch, out_size);
    // the place of four features of a row; behind the buffer's end for what is not in the result
    const auto place = [&](int i, int g, int64_t pitch, int size) {
        const int feature = matmul_four(a, g, q);
        return m + 16 * i + r < a.m && n + feature < a.n ? (16 * i + r) * (int)(pitch * size) + feature * size : (int)0x80000000;
    };
    const bool runs = MB <= 4 && a.out_runs, residual = a.residual && runs;  // larger tiles of whole runs have a kernel of their own
    const auto fetch = [&](int i) {
        v16u row{};
        if (res_size == 4) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4u y = __builtin_amdgcn_raw_buffer_load_b128(from, place(i, g, a.r_pitch, 4), 0, 0);
                row[4 * g] = y[0], row[4 * g + 1] = y[1], row[4 * g + 2] = y[2], row[4 * g + 3] = y[3];
            }
        } else if (fours) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v2u y = __builtin_amdgcn_raw_buffer_load_b64(from, place(i, g, a.r_pitch, 2), 0, 0);
                row[2 * g] = y[0], row[2 * g + 1] = y[1];
            }
        } else {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const v4u y = __builtin_amdgcn_raw_buffer_load_b128(from, place(i, 2 * g, a.r_pitch, 2), 0, 0);
                row[4 * g] = y[0], row[4 * g + 1] = y[1], row[4 * g + 2] = y[2], row[4 * g + 3] = y[3];
            }
        }
        return row;
    };
    v16u now{}, then{};
    if (residual) now = fetch(0);
    float scale[16], bias[16], row_scale[MB];
    const float all = a.w_scales && !a.w_each ? *a.w_scales : 1.0f;
#pragma unroll
    for (int i = 0; i < MB; ++i) row_scale[i] = matmul_row_scale(a, m + 16 * i + r);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int f = n + matmul_four(a, g, q);
        float s[4] = {all, all, all, all}, b[4] = {};
        if (a.w_each && f < a.n) matmul_read(a.w_scales + f, a.n - f, s);
        if (a.bias && f < a.n) matmul_read(a.bias + f, a.n - f, b);
#pragma unroll
        for (int l = 0; l < 4; ++l) scale[4 * g + l] = s[l], bias[4 * g + l] = b[l];
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        if (residual && i + 1 < MB) then = fetch(i + 1);
        float v[16];
#pragma unroll
        for (int l = 0; l < 16; ++l) v[l] = (float)sum[l / 4][i][l % 4] * row_scale[i] * scale[l] + bias[l];
        act_apply<true>(v, a.act);
        if (residual) {
            matmul_typed(a.res_type, [&](auto t) { matmul_add_row<decltype(t)>(now, v); });
            if (a.act2.kind != CLDNN_HIP_ACT_NONE) act_apply<true>(v, a.act2);
            now = then;
        }
        if (runs) {
            matmul_typed(a.out_type, [&](auto t) {
                typedef decltype(t) T;
                constexpr int R = matmul_run(sizeof(T));
                typedef T vec __attribute__((ext_vector_type(R)));
#pragma unroll
                for (int l = 0; l < 16; l += R) {
                    vec x;
#pragma unroll
                    for (int k = 0; k < R; ++k) x[k] = (T)v[l + k];
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x), to, place(i, l / 4, a.o_pitch, sizeof(T)), 0, 0);
                }
            });
            continue;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float x[4] = {v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            matmul_write_row<int8_t>(a, x, m + 16 * i + r, n + matmul_four(a, g, q), out);
        }
    }
}

// The sums of a wave, 16 MB rows from m on x 64 features from n on, of float operands: bias, activation, residual, the result.
template <typename T, int MB>
__device__ __forceinline__ void matmul_finish_rows(const MatmulFloatArgs& a, const v4f (&sum)[4][MB], int m, int n, int lane, void* out)
{
    const int q = lane >> 4, r = lane & 15;
    n += 16 * q;
    float bias[16] = {};
    if (a.bias && n < a.n) matmul_read(a.bias + n, a.n - n, bias);
    act_choose(a.act.kind, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            float v[16];
#pragma unroll
            for (int l = 0; l < 16; ++l) v[l] = sum[l / 4][i][l % 4] + bias[l];
#pragma unroll
            for (int l = 0; l < 16; ++l) v[l] = act_one<decltype(kind)::value>(v[l], a.act.m, a.act.n);
            matmul_write_row<T>(a, v, m + i * 16 + r, n, out);
        }
    });
}

// Which of a wave's 64 features the b-th of its rows of weights is: 16 (r / 4) + 4 t + r % 4 for row 16 t + r.  The four results that the
// matrix instruction leaves in a lane are neighbours, and so are those of the four blocks t: 16 features of one row of the result.
__device__ inline int matmul_feature(const MatmulArgs&, int b) { return 16 * (b >> 2 & 3) + 4 * (b >> 4) + (b & 3); }

// BM x BN of the result to a workgroup of WM x WN waves, 16 MB rows x 64 features to a wave.  Both operands come 64 deep into two LDS
// buffers by direct loads, one step ahead of the one that is multiplied.  A row of 64 values is eight pieces of 16 bytes; piece c
// of row r lies at place c ^ (r >> 1 & 7), so that the sixteen lanes that LDS serves at a time read all of its 64 banks.  Rows
// behind the last are the last one again; pieces behind K are asked for behind the buffer's end, which gives zeros.
// Measured (bf16): 8192 x 8192 x 8192 in 809 to 830 us on several cards, 1.33 to 1.36 PFLOP/s, the library's product 1.40; the matrix
// units are busy in 72 % of the time, at the 1.5 GHz that the power limit leaves.  On the way there: 32x32x16 instructions 882 us,
// both halves of the waves in step 926, tiles of a die in a row instead of a block 959.  25088 x 1024 -> 4096 with a gelu 232 us, its
// product alone 203: seven rounds of 16 steps, 4 us of each the prologue and the stores, 4 the gelu, which nothing overlaps.
template <typename T, int WM, int WN, int MB, int ST, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void matmul_tile_kernel(typename MatmulType<T>::Args a, const T* x, const T* w, void* out)
{
    typedef MatmulType<T> Type;
    typedef typename Type::V V;
    typedef typename Type::Sum Sum;
    constexpr int S = sizeof(T), E = Type::E;
    constexpr int WAVES = WM * WN, BM = WM * MB * 16, BN = WN * 64, BK = 8 * E;
    constexpr int XL = (BM / 8 + WAVES - 1) / WAVES, WL = BN / 8 / WAVES;  // loads of a wave: 8 rows each
    __shared__ v4i lds[KG * ST * (BM + BN) * 8];
    const int lane = threadIdx.x & 63, every = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = every / WAVES, wave = every - group * WAVES;
    const v4i *xt = lds + group * ST * (BM + BN) * 8, *wt = xt + ST * BM * 8;
    const uint32_t xl = lds_address(xt), wl = lds_address(wt);
    const int q = lane >> 4, r = lane & 15;
    int tm, tn;
    matmul_place(a, blockIdx.x, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int steps = ((a.k + BK - 1) / BK + KG - 1) / KG;  // group g takes every KG-th step from the g-th on

    const auto xs = buffer_of(x + (int64_t)m0 * a.a_pitch), ws = buffer_of(w + (int64_t)n0 * a.w_pitch);
    int xo[XL], wo[WL];
    const int turn = lane >> 4;  // row / 2 of the lane's row in a load; loads start at multiples of 8, which count by bit 3 only
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int row = (i * WAVES + wave) * 8 + (lane >> 3);
        xo[i] = min(row, a.m - 1 - m0) * (int)(a.a_pitch * S) + 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int row = (i * WAVES + wave) * 8 + (lane >> 3), b = row & 63;
        const int feature = (row & ~63) + matmul_feature(a, b);
        wo[i] = min(feature, a.n - 1 - n0) * (int)(a.w_pitch * S) + 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
    // every load of a wave starts at the same multiple of 8 modulo 16
    const int piece = (lane & 7) ^ (turn | (wave & 1) << 2);
    static_assert(WAVES % 2 == 0, "");
    const auto load = [&](int step, int at) {
        step = step * KG + group;
        const int behind = step * BK + E * piece >= a.k ? (int)0x80000000 : 0;
#pragma unroll
        for (int i = 0; i < XL; ++i)
            if (BM / 8 % WAVES == 0 || i * WAVES + wave < BM / 8)
                load_lds(xs, xl + at * BM * 128 + (i * WAVES + wave) * 1024, xo[i] | behind, step * S * BK);
#pragma unroll
        for (int i = 0; i < WL; ++i) load_lds(ws, wl + at * BN * 128 + (i * WAVES + wave) * 1024, wo[i] | behind, step * S * BK);
    };
    const int wm = wave / WN, wn = wave - wm * WN;
    Sum acc[4][MB] = {};
    V xf[MB], wf[4];
    const auto read = [&](int round, int at) {
        const int place = (4 * round + q) ^ (r >> 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) wf[j] = __builtin_bit_cast(V, wt[at * BN * 8 + (wn * 64 + j * 16 + r) * 8 + place]);
#pragma unroll
        for (int i = 0; i < MB; ++i) xf[i] = __builtin_bit_cast(V, xt[at * BM * 8 + ((wm * MB + i) * 16 + r) * 8 + place]);
    };
    const auto multiply = [&]() {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][i] = mfma16(wf[j], xf[i], acc[j][i]);
    };
    if constexpr (WAVES == 8) {
        load(0, 0);
        matmul_arrive<0>();
        // The second half of the waves runs one phase behind the first: on every SIMD one wave multiplies while the other fetches
        // its operands.  A step is two rounds of that.
        const bool late = wave >= WAVES / 2;
        if (late) matmul_meet();
        for (int step = 0, at = 0; step < steps; ++step, at ^= 1) {
            load(step + 1, at ^ 1);
            read(0, at);
            matmul_meet();
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
            matmul_meet();
            read(1, at);
            // all reads of this buffer are done and the next step's loads have landed where the late waves end this phase
            if (late) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            matmul_meet();
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
            if (!late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            matmul_meet();
        }
        if (!late) matmul_meet();
    } else {
        // ST - 1 steps under way; what covers a wave's waits is another workgroup on its CU
        static_assert(BM / 8 % WAVES == 0, "as many loads of every wave");
#pragma unroll
        for (int i = 0; i + 1 < ST; ++i) load(i, i);
        for (int step = 0, at = 0, to = ST - 1; step < steps; ++step) {
            matmul_arrive<(ST - 2) * (XL + WL)>();
            load(step + ST - 1, to);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                read(s, at);
                multiply();
            }
            to = at;
            at = at + 1 == ST ? 0 : at + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if constexpr (KG > 1) {
        // the groups' sums meet in LDS, in the order of the groups: group g finishes every KG-th block of rows
        static_assert(KG * WAVES * MB * 256 <= KG * ST * (BM + BN) * 8 && (KG - 1) * MB >= 1, "the sums fit where the operands were");
        asm volatile("s_barrier" ::: "memory");
        Sum* sums = (Sum*)lds;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[(((group * WAVES + wave) * MB + i) * 4 + j) * 64 + lane] = acc[j][i];
        __syncthreads();
        for (int i = group; i < MB; i += KG) {
            Sum sum[4][1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sum[j][0] = sums[((wave * MB + i) * 4 + j) * 64 + lane];
#pragma unroll
                for (int g = 1; g < KG; ++g) sum[j][0] += sums[(((g * WAVES + wave) * MB + i) * 4 + j) * 64 + lane];
            }
            const int m = m0 + (wm * MB + i) * 16, n = n0 + wn * 64;
            if constexpr (E == 16) matmul_finish_s8(a, sum, m, n, lane, out);
            else matmul_finish_rows<T>(a, sum, m, n, lane, out);
        }
    } else {
        const int m = m0 + wm * MB * 16, n = n0 + wn * 64;
        if constexpr (E == 16) matmul_finish_s8(a, acc, m, n, lane, out);
        else matmul_finish_rows<T>(a, acc, m, n, lane, out);
    }
}

// Operands whose rows are no whole 16-byte pieces, copied into rows that are, zeros behind K: row i of a, then row j of weights.
template <typename T>
__global__ __launch_bounds__(MATMUL_PACK_THREADS) void matmul_pack_kernel(MatmulArgs a, const T* x, const T* w, v4i* to, int pieces)
{
    const int64_t i = (int64_t)blockIdx.x * MATMUL_PACK_THREADS + threadIdx.x, row = i / pieces;
    const int k = (int)(i - row * pieces) * MatmulType<T>::E;
    if (row >= a.m + a.n) return;
    to[i] = matmul_load(row < a.m ? x + row * a.a_pitch : w + (row - a.m) * a.w_pitch, k, a.k);
}

}  // namespace chip
