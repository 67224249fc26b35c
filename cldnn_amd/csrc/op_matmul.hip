// Matrix product with bias, activation and residual: out = act2(act(a w^T + bias) + residual).
//
// The weights are the row operand of the matrix instruction, so that a lane ends with neighbouring features of one row of the
// result: whole 16-byte stores, and a bias and a residual that are read the same way.
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
    int32_t band;                     // rows of tiles in a band
    int32_t splits;                   // workgroups that split K for each tile: their sums go to part[split][m][n]
    float* part;
};

constexpr int64_t MATMUL_PACK = 200ll << 20;  // products from which unaligned operands are copied
constexpr int MATMUL_PACK_THREADS = 256;

struct MatmulPlan {
    MatmulArgs a;
    int dt;
    int kernel;  // row of matmul_kernels; the one for any strides where pointers are not aligned
    int any;
    int pieces;  // > 0: the operands are copied into rows of so many 16-byte pieces first
};

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
__device__ __forceinline__ void matmul_read(const R* p, int valid, float (&v)[N])
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
__device__ __forceinline__ void matmul_write(O* p, int valid, const float (&v)[N])
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
__device__ __forceinline__ void matmul_write_row(const MatmulArgs& a, float (&v)[N], int m, int n0, void* out)
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
// -> 4096 39 us, 5.3 TB/s, a large copy's rate; with 16 rows 55 us, their values being as many bytes again from the die's L2.
template <typename T, int FT, int PT, int U, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void matmul_split_kernel(MatmulArgs a, const T* x, const T* w, void* out)
{
    typedef typename vec8<T>::type V;
    constexpr int TILE = 256 * FT * PT;
    __shared__ float sums[WAVES][TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    int tm, tn;
    matmul_place(a, blockIdx.x, tm, tn);
    const int m0 = tm * 16 * PT, n0 = tn * 16 * FT;
    const T *xr[PT], *wr[FT];
#pragma unroll
    for (int i = 0; i < PT; ++i) xr[i] = x + (int64_t)min(m0 + 16 * i + r, a.m - 1) * a.a_pitch + 8 * q;
#pragma unroll
    for (int i = 0; i < FT; ++i) wr[i] = w + (int64_t)min(n0 + 16 * i + r, a.n - 1) * a.w_pitch + 8 * q;
    v4f acc[FT][PT] = {};
    const int whole = a.k / (32 * U);  // runs of U full steps, dealt to the waves in turn
    const int worker = blockIdx.y * WAVES + wave, workers = a.splits * WAVES;
    for (int run = worker; run < whole; run += workers) {
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
    const int steps = a.k / 32 + (a.k % 32 != 0);
    for (int step = whole * U + (worker - whole % workers + workers) % workers; step < steps; step += workers) {
        const int k = step * 32;
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
        const int row = at / (16 * FT), n = n0 + at - row * 16 * FT;
        if (a.splits > 1) {
            if (m0 + row < a.m && n < a.n) matmul_write(a.part + ((int64_t)blockIdx.y * a.m + m0 + row) * a.n + n, a.n - n, v);
            continue;
        }
        if (a.bias && n < a.n) {
            float b[N];
            matmul_read(a.bias + n, a.n - n, b);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += b[i];
        }
        act_apply(v, a.act);
        matmul_write_row<T>(a, v, m0 + row, n, out);
    }
}

// The sums of the workgroups that split K, joined in their order: four features of a row to a thread.
template <typename T>
__global__ __launch_bounds__(256) void matmul_join_kernel(MatmulArgs a, void* out)
{
    const int across = (a.n + 3) / 4, i = blockIdx.x * 256 + threadIdx.x, m = i / across, n = (i - m * across) * 4;
    if (m >= a.m) return;
    float v[4];
    matmul_read(a.part + (int64_t)m * a.n + n, a.n - n, v);
#pragma unroll 4
    for (int s = 1; s < a.splits; ++s) {
        float x[4];
        matmul_read(a.part + ((int64_t)s * a.m + m) * a.n + n, a.n - n, x);
#pragma unroll
        for (int l = 0; l < 4; ++l) v[l] += x[l];
    }
    if (a.bias) {
        float b[4];
        matmul_read(a.bias + n, a.n - n, b);
#pragma unroll
        for (int l = 0; l < 4; ++l) v[l] += b[l];
    }
    act_apply(v, a.act);
    matmul_write_row<T>(a, v, m, n, out);
}

// BM x BN of the result to a workgroup of WM x WN waves, 16 MB rows x 64 features to a wave.  Both operands come 64 deep into two LDS
// buffers by direct loads, one step ahead of the one that is multiplied.  A row of 64 values is eight pieces of 16 bytes; piece c
// of row r lies at place c ^ (r >> 1 & 7), so that the sixteen lanes that LDS serves at a time read all of its 64 banks.  Rows
// behind the last are the last one again; pieces behind K are asked for behind the buffer's end, which gives zeros.
// Measured (bf16): 8192 x 8192 x 8192 in 809 to 830 us on several cards, 1.33 to 1.36 PFLOP/s, the library's product 1.40; the matrix
// units are busy in 72 % of the time, at the 1.5 GHz that the power limit leaves.  On the way there: 32x32x16 instructions 882 us,
// both halves of the waves in step 926, tiles of a die in a row instead of a block 959.  25088 x 1024 -> 4096 with a gelu 232 us, its
// product alone 203: seven rounds of 16 steps, 4 us of each the prologue and the stores, 4 the gelu, which nothing overlaps.
// Row 16 t + r of a wave's 64 rows of weights is feature 16 (r / 4) + 4 t + r % 4 of its 64: the four results that the matrix
// instruction leaves in a lane are neighbours, and so are those of the four blocks t: 16 features of one row of the result.
template <typename T, int WM, int WN, int MB, int ST, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void matmul_tile_kernel(MatmulArgs a, const T* x, const T* w, void* out)
{
    typedef typename vec8<T>::type V;
    constexpr int WAVES = WM * WN, BM = WM * MB * 16, BN = WN * 64, BK = 64;
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
        xo[i] = min(row, a.m - 1 - m0) * (int)(a.a_pitch * 2) + 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int row = (i * WAVES + wave) * 8 + (lane >> 3), b = row & 63;
        const int feature = (row & ~63) + 16 * (b >> 2 & 3) + 4 * (b >> 4) + (b & 3);
        wo[i] = min(feature, a.n - 1 - n0) * (int)(a.w_pitch * 2) + 16 * ((lane & 7) ^ (row >> 1 & 7));
    }
    // every load of a wave starts at the same multiple of 8 modulo 16
    const int piece = (lane & 7) ^ (turn | (wave & 1) << 2);
    static_assert(WAVES % 2 == 0, "");
    const auto load = [&](int step, int at) {
        step = step * KG + group;
        const int behind = step * BK + 8 * piece >= a.k ? (int)0x80000000 : 0;
#pragma unroll
        for (int i = 0; i < XL; ++i)
            if (BM / 8 % WAVES == 0 || i * WAVES + wave < BM / 8)
                load_lds(xs, xl + at * BM * 128 + (i * WAVES + wave) * 1024, xo[i] | behind, step * 2 * BK);
#pragma unroll
        for (int i = 0; i < WL; ++i) load_lds(ws, wl + at * BN * 128 + (i * WAVES + wave) * 1024, wo[i] | behind, step * 2 * BK);
    };
    const int wm = wave / WN, wn = wave - wm * WN;
    v4f acc[4][MB] = {};
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
    const int n = n0 + wn * 64 + 16 * q;
    if constexpr (KG > 1) {
        // the groups' sums meet in LDS, in the order of the groups: group g finishes every KG-th block of rows
        static_assert(KG * WAVES * MB * 256 <= KG * ST * (BM + BN) * 8 && (KG - 1) * MB >= 1, "the sums fit where the operands were");
        asm volatile("s_barrier" ::: "memory");
        v4f* sums = (v4f*)lds;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[(((group * WAVES + wave) * MB + i) * 4 + j) * 64 + lane] = acc[j][i];
        __syncthreads();
        for (int i = group; i < MB; i += KG) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v4f t = sums[((wave * MB + i) * 4 + j) * 64 + lane];
#pragma unroll
                for (int g = 1; g < KG; ++g) t += sums[(((g * WAVES + wave) * MB + i) * 4 + j) * 64 + lane];
#pragma unroll
                for (int l = 0; l < 4; ++l) v[4 * j + l] = t[l];
            }
            float bias[16] = {};
            if (a.bias && n < a.n) matmul_read(a.bias + n, a.n - n, bias);
#pragma unroll
            for (int l = 0; l < 16; ++l) v[l] += bias[l];
            act_apply(v, a.act);
            matmul_write_row<T>(a, v, m0 + (wm * MB + i) * 16 + r, n, out);
        }
    } else {
        float bias[16] = {};
        if (a.bias && n < a.n) matmul_read(a.bias + n, a.n - n, bias);
        act_choose(a.act.kind, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                float v[16];
#pragma unroll
                for (int l = 0; l < 16; ++l) v[l] = acc[l / 4][i][l % 4] + bias[l];
#pragma unroll
                for (int l = 0; l < 16; ++l) v[l] = act_one<decltype(kind)::value>(v[l], a.act.m, a.act.n);
                matmul_write_row<T>(a, v, m0 + (wm * MB + i) * 16 + r, n, out);
            }
        });
    }
}

// Operands whose rows are no whole 16-byte pieces, copied into rows that are, zeros behind K: row i of a, then row j of weights.
template <typename T>
__global__ __launch_bounds__(MATMUL_PACK_THREADS) void matmul_pack_kernel(MatmulArgs a, const T* x, const T* w, v4i* to, int pieces)
{
    const int64_t i = (int64_t)blockIdx.x * MATMUL_PACK_THREADS + threadIdx.x, row = i / pieces;
    const int k = (int)(i - row * pieces) * 8;
    if (row >= a.m + a.n) return;
    to[i] = matmul_load8(row < a.m ? x + row * a.a_pitch : w + (row - a.m) * a.w_pitch, k, a.k);
}

struct MatmulKernel {
    const char* name;
    int rows, features, waves;
    int lds;  // bytes: the stages of both operands, or the waves' sums
};
enum { MM_256, MM_224, MM_192, MM_128, MM_64x128, MM_64, MM_32, MM_ANY_64, MM_ANY_32, MM_16 };
static const MatmulKernel matmul_kernels[] = {
    {"matmul_tile<256x256>", 256, 256, 8, 128 << 10}, {"matmul_tile<224x256>", 224, 256, 8, 120 << 10}, {"matmul_tile<192x256>", 192, 256, 8, 112 << 10},
    {"matmul_tile<128x128>", 128, 128, 4, 64 << 10}, {"matmul_tile<64x128>", 64, 128, 4, 72 << 10},
    {"matmul_tile<64x64,k2>", 64, 64, 8, 128 << 10}, {"matmul_tile<32x64,k4>", 32, 64, 8, 144 << 10},
    {"matmul_split<64x64>", 64, 64, 4, 64 << 10}, {"matmul_split<32x32>", 32, 32, 8, 32 << 10}, {"matmul_split<16x16>", 16, 16, 8, 8 << 10},
};

static int64_t matmul_pack_blocks(const MatmulPlan& p) { return (((int64_t)p.a.m + p.a.n) * p.pieces + MATMUL_PACK_THREADS - 1) / MATMUL_PACK_THREADS; }

static int64_t matmul_count(int m, int n, const MatmulKernel& k) { return (int64_t)((m + k.rows - 1) / k.rows) * ((n + k.features - 1) / k.features); }

// whole: rows of 16-byte pieces, which the direct loads into LDS need
static int matmul_choose(int m, int n, bool whole, int cus)
{
    const auto tiles = [&](int row) { return matmul_count(m, n, matmul_kernels[row]); };
    const auto rounds = [&](int row) { return (tiles(row) + cus - 1) / cus; };
    // Few tiles of any size: the smallest, whose eight waves split K.  (us, against 32 x 64 tiles: 1 x 2048 -> 1000 4.7 and 7.0, 64 x 2048
    // -> 1000 6.0 and 7.0; at twice as many tiles, 32 x 1024 -> 4096, 6.0 and 5.2.  The bound is that of such K; at 8192 it is late: 16 x
    // 8192 -> 5120, 320 of them, 30.7, -> 5136 in 32 x 64 tiles 17.6)
    if (tiles(MM_16) * 4 <= cus * 5) return MM_16;
    if (!whole) return tiles(MM_ANY_64) >= cus ? MM_ANY_64 : MM_ANY_32;
    if (tiles(MM_128) * 4 >= cus * 5) {
        // A CU's time by the rows of its 256 features, which the smaller tiles fetch more operands for: measured at 8192 x 8192 x
        // 8192, per row of a round, 1 / 1.02 / 1.11 / 1.22 (809 us, 902, 1010, 991).  25088 x 4096 -> 1024: 222, 210, 287 and 268 us.
        const int kernel[] = {MM_256, MM_224, MM_192, MM_128};
        const double time[] = {rounds(MM_256) * 256.0, rounds(MM_224) * 224 * 1.04, rounds(MM_192) * 192 * 1.12, rounds(MM_128) * 64 * 1.22};
        return kernel[std::min_element(time, time + 4) - time];
    }
    // Fewer: what leaves no CU idle and pays the fewest trips to memory one behind the other.  (3136 x 512 -> 512: 128 x 128 8.8 us,
    // 64 x 128 6.1, 64 x 64 9.1; 1024 x 1024 -> 1024: 13.3, 8.3, 6.6, 32 x 64 10.1; 196 x 1024 -> 2048: 12.3, 8.1, 6.2, 5.2)
    if (tiles(MM_64x128) * 4 >= cus * 3) return MM_64x128;
    if (tiles(MM_64) * 4 >= cus * 3) return MM_64;
    return MM_32;
}

static void matmul_tiles(MatmulArgs& a, const MatmulKernel& k)
{
    const int64_t tiles = matmul_count(a.m, a.n, k);
    check_grid(tiles, 64 * k.waves, "matmul");
    a.tiles = (int32_t)tiles, a.tiles_m = (a.m + k.rows - 1) / k.rows, a.tiles_n = (a.n + k.features - 1) / k.features;
    a.band = 8;
}

MatmulPlan* matmul_plan(const cldnn_hip_engine_s& e, const cldnn_hip_matmul_desc& d, cldnn_hip_operator_info& info)
{
    const auto is_half = [](int dt) { return dt == CLDNN_HIP_F16 || dt == CLDNN_HIP_BF16; };
    CHIP_REQUIRE(d.m > 0 && d.n > 0 && d.k > 0, CLDNN_HIP_INVALID_ARG, "matmul: sizes must be positive");
    // so that a tile's last row or feature, and a step's last value, has a number
    CHIP_REQUIRE(std::max(d.m, std::max(d.n, d.k)) <= INT32_MAX - 256, CLDNN_HIP_UNSUPPORTED_SIZE, "matmul: too large");
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
    const bool whole = d.k % 8 == 0 && a.a_pitch % 8 == 0 && a.w_pitch % 8 == 0 && std::max(a.a_pitch, a.w_pitch) < (1 << 21);
    plan->kernel = matmul_choose(d.m, d.n, whole, cus);
    plan->any = matmul_choose(d.m, d.n, false, cus);
    // The copy costs a launch and two trips of the operands, the kernels for any rows 5 times the tiles' time from there on (4000 x 255
    // -> 1000: 41 us without it, 10 with).
    if (!whole && plan->any != MM_16 && d.k < (1 << 20) && (double)d.m * d.n * d.k >= MATMUL_PACK && ((int64_t)d.m + d.n) * ((d.k + 7) / 8) < (1ll << 32) - MATMUL_PACK_THREADS) {
        plan->pieces = (d.k + 7) / 8;
        plan->kernel = matmul_choose(d.m, d.n, true, cus);
    }
    const MatmulKernel& kernel = matmul_kernels[plan->kernel];
    matmul_tiles(a, kernel);
    // The smallest tiles that leave half of the chip idle over a long K: several workgroups to a tile, for the price of a second launch.
    // Without it and with it: 16 x 1000 x 25088 44.9 and 20.3 us, 1 x 500 x 25088 29.0 and 10.8, 8 x 1000 x 16384 24.9 and 12.4,
    // 4 x 2000 x 8000 12.5 and 11.6; 1 x 1000 x 4096 6.6 and 9.3, so from 8000 on.  Beyond half of the chip it is not done, and the step
    // shows: 16 x 2048 x 25088, 128 tiles of two workgroups, 31.4 us, 16 x 2064 x 25088, 129 of one, 50.8.
    a.splits = 1;
    if (plan->kernel == MM_16 && a.tiles * 2 <= cus && d.k >= 8000) a.splits = std::min(cus / a.tiles, d.k / 2048);
    info.launches = plan->pieces || a.splits > 1 ? 2 : 1, info.block = 64 * kernel.waves, info.grid = a.tiles * a.splits, info.lds_bytes = kernel.lds;
    if (plan->pieces) info.block = MATMUL_PACK_THREADS, info.grid = (int32_t)matmul_pack_blocks(*plan);
    info.workspace_bytes = ((int64_t)d.m + d.n) * plan->pieces * 16 + (a.splits > 1 ? (int64_t)a.splits * d.m * d.n * 4 : 0);
    info.ops = 2ll * d.m * d.n * d.k;
    info.bytes = 2 * ((int64_t)d.m * d.k + (int64_t)d.n * d.k) + (d.has_bias ? 4ll * d.n : 0) + (int64_t)d.m * d.n * (out_size + res_size);
    snprintf(info.kernel_name, sizeof info.kernel_name, "%s%s%s", plan->pieces ? "matmul_pack + " : "", kernel.name, a.splits > 1 ? " + matmul_join" : "");
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
        const void *xa = x, *wa = w;
        a.part = (float*)workspace;
        if (p.pieces) {
            hipLaunchKernelGGL((matmul_pack_kernel<T>), dim3((unsigned)matmul_pack_blocks(p)), dim3(MATMUL_PACK_THREADS), 0, s, a, (const T*)x, (const T*)w, (v4i*)workspace, p.pieces);
            a.a_pitch = a.w_pitch = a.k = 8 * p.pieces;
            xa = workspace, wa = (const v4i*)workspace + (int64_t)a.m * p.pieces;
        }
        const int row = (((uintptr_t)xa | (uintptr_t)wa) & 15) == 0 ? p.kernel : p.any;
        const MatmulKernel& kernel = matmul_kernels[row];
        matmul_tiles(a, kernel);
        const auto launch = [&](auto f) { hipLaunchKernelGGL(f, dim3(a.tiles, a.splits), dim3(64 * kernel.waves), 0, s, a, (const T*)xa, (const T*)wa, out); };
        switch (row) {
        case MM_256: launch(matmul_tile_kernel<T, 2, 4, 8, 2, 1>); break;
        case MM_224: launch(matmul_tile_kernel<T, 2, 4, 7, 2, 1>); break;
        case MM_192: launch(matmul_tile_kernel<T, 2, 4, 6, 2, 1>); break;
        case MM_128: launch(matmul_tile_kernel<T, 2, 2, 4, 2, 1>); break;
        case MM_64x128: launch(matmul_tile_kernel<T, 2, 2, 2, 3, 1>); break;
        case MM_64: launch(matmul_tile_kernel<T, 4, 1, 1, 4, 2>); break;
        case MM_32: launch(matmul_tile_kernel<T, 2, 1, 1, 3, 4>); break;
        case MM_ANY_64: launch(matmul_split_kernel<T, 4, 4, 2, 4>); break;
        case MM_ANY_32: launch(matmul_split_kernel<T, 2, 2, 4, 8>); break;
        default: launch(matmul_split_kernel<T, 1, 1, 16, 8>);
        }
        if (a.splits > 1)
            hipLaunchKernelGGL((matmul_join_kernel<T>), dim3((unsigned)(((int64_t)a.m * ((a.n + 3) / 4) + 255) / 256)), dim3(256), 0, s, a, out);
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(MatmulPlan* p) { delete p; }

}  // namespace chip
