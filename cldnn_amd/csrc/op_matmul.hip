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
    int32_t tiles, tiles_m, tiles_n;  // of the result
    int32_t by_rows;                  // neighbouring tiles share their rows; otherwise their features
};

struct MatmulPlan {
    MatmulArgs a;
    int dt;
    int kernel;  // row of matmul_kernels; the one for any strides where pointers are not aligned
    int any;
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

template <typename R, int N>
__device__ inline void matmul_read(const R* p, int valid, float (&v)[N])
{
    if (valid >= N) {
        constexpr int W = 16 / sizeof(R) < N ? 16 / sizeof(R) : N;
        typedef R any __attribute__((ext_vector_type(W), aligned(sizeof(R))));
#pragma unroll
        for (int i = 0; i < N / W; ++i) {
            const any x = ((const any*)p)[i];
#pragma unroll
            for (int j = 0; j < W; ++j) v[W * i + j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? (float)p[i] : 0.0f;
    }
}

template <typename O, int N>
__device__ inline void matmul_write(O* p, int valid, const float (&v)[N])
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

// N neighbouring features from n0 on of row m
template <typename T, int N>
__device__ inline void matmul_finish(const MatmulArgs& a, float (&v)[N], int m, int n0, void* out)
{
    const int valid = a.n - n0;
    if (m >= a.m || valid <= 0) return;
    if (a.bias) {
        float b[N];
        matmul_read(a.bias + n0, valid, b);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += b[i];
    }
    act_apply(v, a.act);
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

// Tiles are dealt to the accelerator dies in turn (workgroup i runs on die i % 8): each die gets a run of neighbouring tiles, whose
// operands its own L2 then serves.
__device__ inline int matmul_tile(const MatmulArgs& a, int i)
{
    const int die = i & 7, each = a.tiles >> 3, more = a.tiles & 7;
    return die * each + min(die, more) + (i >> 3);
}

__device__ inline __amdgpu_buffer_rsrc_t matmul_rsrc(const void* p)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7fffffff, 0x00020000);
}

// lane t's 16 bytes at `offset` + `step` go to LDS at place t from `to` on
__device__ inline void matmul_load_lds(__amdgpu_buffer_rsrc_t from, v4i* to, int offset, int step)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, offset, step, 0, 0);
}

// all of this wave's loads have landed, then every wave's
__device__ inline void matmul_arrive()
{
    // by builtins: the compiler knows then that nothing is under way, and waits for no loads of its own accord behind it
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // loads have landed, LDS reads are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Few rows, or few tiles: 16 FT features x 16 PT rows to a workgroup, whose waves split K; both operands straight from memory into
// the registers that the matrix instruction reads, U steps of 32 at a time; the partial sums meet in LDS.
template <typename T, int FT, int PT, int U, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void matmul_split_kernel(MatmulArgs a, const T* x, const T* w, void* out)
{
    typedef typename vec8<T>::type V;
    constexpr int TILE = 256 * FT * PT;
    __shared__ float sums[WAVES][TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int tile = matmul_tile(a, blockIdx.x);
    const int tm = a.by_rows ? tile / a.tiles_n : tile % a.tiles_m, tn = a.by_rows ? tile % a.tiles_n : tile / a.tiles_m;
    const int m0 = tm * 16 * PT, n0 = tn * 16 * FT;
    const T *xr[PT], *wr[FT];
#pragma unroll
    for (int i = 0; i < PT; ++i) xr[i] = x + (int64_t)min(m0 + 16 * i + r, a.m - 1) * a.a_pitch + 8 * q;
#pragma unroll
    for (int i = 0; i < FT; ++i) wr[i] = w + (int64_t)min(n0 + 16 * i + r, a.n - 1) * a.w_pitch + 8 * q;
    v4f acc[FT][PT] = {};
    const int whole = a.k / (32 * U);  // runs of U full steps, dealt to the waves in turn
    for (int run = wave; run < whole; run += WAVES) {
        const int k = run * 32 * U;
        v4i wf[U][FT], xf[U][PT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < FT; ++i) wf[u][i] = *(const v4i_any*)(wr[i] + k + 32 * u);
#pragma unroll
            for (int i = 0; i < PT; ++i) xf[u][i] = *(const v4i_any*)(xr[i] + k + 32 * u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int j = 0; j < PT; ++j) acc[i][j] = mfma16(__builtin_bit_cast(V, wf[u][i]), __builtin_bit_cast(V, xf[u][j]), acc[i][j]);
    }
    // the steps behind the runs, one to a wave
    for (int k = whole * 32 * U + 32 * ((wave - whole % WAVES + WAVES) % WAVES); k < a.k; k += 32 * WAVES) {
        v4i wf[FT], xf[PT];
#pragma unroll
        for (int i = 0; i < FT; ++i) wf[i] = matmul_load8(wr[i] - 8 * q, k + 8 * q, a.k);
#pragma unroll
        for (int i = 0; i < PT; ++i) xf[i] = matmul_load8(xr[i] - 8 * q, k + 8 * q, a.k);
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int j = 0; j < PT; ++j) acc[i][j] = mfma16(__builtin_bit_cast(V, wf[i]), __builtin_bit_cast(V, xf[j]), acc[i][j]);
    }
    // [row][feature], so that a thread's N values are neighbouring features
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < PT; ++j) *(v4f*)&sums[wave][(16 * j + r) * 16 * FT + 16 * i + 4 * q] = acc[i][j];
    __syncthreads();
    constexpr int N = TILE / (64 * WAVES) < 1 ? 1 : TILE / (64 * WAVES) > 16 ? 16 : TILE / (64 * WAVES);
    static_assert(16 * FT % N == 0, "a thread's values lie in one row");
    for (int at = threadIdx.x * N; at < TILE; at += 64 * WAVES * N) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = sums[0][at + i];
#pragma unroll
        for (int s = 1; s < WAVES; ++s)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += sums[s][at + i];
        const int row = at / (16 * FT);
        matmul_finish<T>(a, v, m0 + row, n0 + at - row * 16 * FT, out);
    }
}

// BM x BN of the result to a workgroup of WM x WN waves, MB x NB blocks of 32 x 32 to a wave; both operands come 64 deep into two
// LDS buffers by direct loads, the next step's while one is multiplied: one barrier a step.  A row of 64 values is eight pieces
// of 16 bytes; piece c of row r lies at place c ^ (r & 7), so that the eight lanes that LDS serves at a time read eight places.
// Rows behind the last are the last one again; pieces behind K are asked for behind the buffer's end, which gives zeros.
template <typename T, int WM, int WN, int MB, int NB>
__global__ __launch_bounds__(64 * WM * WN) void matmul_tile_kernel(MatmulArgs a, const T* x, const T* w, void* out)
{
    typedef typename vec8<T>::type V;
    constexpr int WAVES = WM * WN, BM = WM * MB * 32, BN = WN * NB * 32;
    constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // loads of a wave: 8 rows each
    __shared__ v4i x0[BM * 8], x1[BM * 8], w0[BN * 8], w1[BN * 8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, r = lane & 31;
    const int tile = matmul_tile(a, blockIdx.x);
    const int tm = a.by_rows ? tile / a.tiles_n : tile % a.tiles_m, tn = a.by_rows ? tile % a.tiles_n : tile / a.tiles_m;
    const int m0 = tm * BM, n0 = tn * BN;
    const int steps = (a.k + 63) / 64, last = a.k - (steps - 1) * 64;  // values of the last step

    const auto xs = matmul_rsrc(x + (int64_t)m0 * a.a_pitch), ws = matmul_rsrc(w + (int64_t)n0 * a.w_pitch);
    int xo[XL], wo[WL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int row = (wave * XL + i) * 8 + (lane >> 3), c = (lane & 7) ^ (row & 7);
        xo[i] = min(row, a.m - 1 - m0) * (int)(a.a_pitch * 2) + 16 * c;
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        // row q of LDS has the feature that row q of the matrix instruction stands for
        const int row = (wave * WL + i) * 8 + (lane >> 3), c = (lane & 7) ^ (row & 7);
        wo[i] = min((row & ~31) + matmul_feature(row & 31), a.n - 1 - n0) * (int)(a.w_pitch * 2) + 16 * c;
    }
    const int reach = 8 * ((lane & 7) ^ (lane >> 3));  // the first of this lane's eight values of a step: (row & 7) == lane >> 3
    const auto load = [&](int step, v4i* xb, v4i* wb) {
        const int behind = step == steps - 1 && reach >= last ? (int)0x80000000 : 0;
#pragma unroll
        for (int i = 0; i < XL; ++i) matmul_load_lds(xs, xb + (wave * XL + i) * 64, xo[i] | behind, step * 128);
#pragma unroll
        for (int i = 0; i < WL; ++i) matmul_load_lds(ws, wb + (wave * WL + i) * 64, wo[i] | behind, step * 128);
    };
    const int wm = wave / WN, wn = wave - wm * WN;
    v16f acc[NB][MB] = {};
    const auto multiply = [&](const v4i* xb, const v4i* wb) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int place = (2 * s + half) ^ (r & 7);
            V xf[MB], wf[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) wf[j] = __builtin_bit_cast(V, wb[((wn * NB + j) * 32 + r) * 8 + place]);
#pragma unroll
            for (int i = 0; i < MB; ++i) xf[i] = __builtin_bit_cast(V, xb[((wm * MB + i) * 32 + r) * 8 + place]);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[j][i] = mfma32(wf[j], xf[i], acc[j][i]);
        }
    };
    load(0, x0, w0);
    for (int step = 0; step < steps; step += 2) {
        matmul_arrive();
        if (step + 1 < steps) load(step + 1, x1, w1);
        multiply(x0, w0);
        if (step + 1 == steps) break;
        matmul_arrive();
        if (step + 2 < steps) load(step + 2, x0, w0);
        multiply(x1, w1);
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float v[16];
#pragma unroll
            for (int l = 0; l < 16; ++l) v[l] = acc[j][i][l];
            matmul_finish<T>(a, v, m0 + (wm * MB + i) * 32 + r, n0 + (wn * NB + j) * 32 + 16 * half, out);
        }
}

struct MatmulKernel {
    const char* name;
    int rows, features, waves;
};
static const MatmulKernel matmul_kernels[] = {
    {"matmul_tile<256x256>", 256, 256, 8}, {"matmul_tile<128x128>", 128, 128, 4},
    {"matmul_split<64x64>", 64, 64, 4}, {"matmul_split<64x32>", 64, 32, 8}, {"matmul_split<32x32>", 32, 32, 8},
    {"matmul_split<64x16>", 64, 16, 8}, {"matmul_split<32x16>", 32, 16, 16}, {"matmul_split<16x16>", 16, 16, 16},
};

static int64_t matmul_count(int m, int n, const MatmulKernel& k) { return (int64_t)((m + k.rows - 1) / k.rows) * ((n + k.features - 1) / k.features); }

// whole: rows of 16-byte pieces, which the direct loads into LDS need
static int matmul_choose(int m, int n, int k, bool whole, int cus)
{
    const auto full = [&](int row) { return matmul_count(m, n, matmul_kernels[row]) >= cus; };
    if (whole && full(0)) return 0;
    if (whole && full(1)) return 1;
    if (full(2)) return 2;
    if (m <= 16) return 7;
    if (m <= 32) return 6;
    if (full(3)) return 3;
    if (m > 64 || full(4)) return 4;
    return 5;
}

static void matmul_tiles(MatmulArgs& a, const MatmulKernel& k)
{
    const int64_t tiles = matmul_count(a.m, a.n, k);
    CHIP_REQUIRE(tiles < (1ll << 31), CLDNN_HIP_UNSUPPORTED_SIZE, "matmul: too large");
    a.tiles = (int32_t)tiles, a.tiles_m = (a.m + k.rows - 1) / k.rows, a.tiles_n = (a.n + k.features - 1) / k.features;
    // neighbouring tiles share what is larger
    a.by_rows = a.m >= a.n;
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
    const int cus = e.props.multiProcessorCount;
    plan->kernel = matmul_choose(d.m, d.n, d.k, d.k % 8 == 0 && a.a_pitch % 8 == 0 && a.w_pitch % 8 == 0 && std::max(a.a_pitch, a.w_pitch) < (1 << 21), cus);
    plan->any = matmul_choose(d.m, d.n, d.k, false, cus);
    const MatmulKernel& kernel = matmul_kernels[plan->kernel];
    matmul_tiles(a, kernel);
    info.launches = 1, info.block = 64 * kernel.waves, info.grid = a.tiles;
    info.ops = 2ll * d.m * d.n * d.k;
    info.bytes = 2 * ((int64_t)d.m * d.k + (int64_t)d.n * d.k) + (d.has_bias ? 4ll * d.n : 0) + (int64_t)d.m * d.n * (out_size + res_size);
    snprintf(info.kernel_name, sizeof info.kernel_name, "%s", kernel.name);
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
        const int row = (((uintptr_t)x | (uintptr_t)w) & 15) == 0 ? p.kernel : p.any;
        const MatmulKernel& kernel = matmul_kernels[row];
        matmul_tiles(a, kernel);
        const auto launch = [&](auto f) { hipLaunchKernelGGL(f, dim3(a.tiles), dim3(64 * kernel.waves), 0, s, a, (const T*)x, (const T*)w, out); };
        switch (row) {
        case 0: launch(matmul_tile_kernel<T, 2, 4, 4, 2>); break;
        case 1: launch(matmul_tile_kernel<T, 2, 2, 2, 2>); break;
        case 2: launch(matmul_split_kernel<T, 4, 4, 2, 4>); break;
        case 3: launch(matmul_split_kernel<T, 2, 4, 3, 8>); break;
        case 4: launch(matmul_split_kernel<T, 2, 2, 4, 8>); break;
        case 5: launch(matmul_split_kernel<T, 1, 4, 4, 8>); break;
        case 6: launch(matmul_split_kernel<T, 1, 2, 5, 16>); break;
        default: launch(matmul_split_kernel<T, 1, 1, 8, 16>);
        }
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(MatmulPlan* p) { delete p; }

}  // namespace chip
