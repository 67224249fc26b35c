// Matrix product of int8 operands with scales for each row and channel: out = act2(act(a w^T * row * channel + bias) + residual).
// The kernels are those of the float products (matmul_kernel.h): a row of either type is the same pieces of 16 bytes.
#include "matmul_kernel.h"
#include "ops_s8.h"

namespace chip {

constexpr int MATMUL_S8_MOST_K = 131071;  // 128 * 128 of each fit 31 bits
constexpr int64_t MATMUL_S8_PAST = 64 << 20;  // twice what the dies' caches hold together
constexpr int64_t MATMUL_S8_RUN_PITCH = 1 << 20;  // 256 rows of it in f32 are within a buffer's reach
// Products from which unaligned operands are copied: a launch and two trips of the operands against the kernels for any rows (us, without
// the copy and with it: 1000 x 401 -> 400 7.1 and 7.9, 1000 x 255 -> 1000 9.2 and 8.1, 1500 x 255 -> 1000 13.0 and 8.4, 20000 x 84 -> 400
// 27 and 12).
constexpr int64_t MATMUL_S8_PACK = 200ll << 20;

// Large products: 32 MB rows x 256 features at a time to a workgroup of 2 x 4 waves, which goes through tiles i, i + grid, .. of the result.
// The main loop is that of matmul_tile_kernel<2, 4, MB>, whose comment says how the halves of the waves take turns; what is different
// is the end of a tile.  The next tile's first operands are asked for in front of it, and its stores drain under the next one's products,
// where a workgroup to a tile waits for all of them before its LDS is free for the next.  Scales and bias are asked for a tile ahead,
// a value to a thread, and handed out through LDS; every place of the result is an offset that is worked out once.
// Bound by the matrix cores at the power limit, and by the end of a tile in the vector units (on several cards, 8192 x 8192 x 8192 419 to
// 445 us, 2.47 to 2.63 POP/s, the matrix cores 63 % of the time busy at 1.97 GHz; 25088 x 1024 -> 4096 with a gelu, eight steps of K to a tile
// and seven rounds of tiles, 127 to 136 us, 1.55 to 1.66 POP/s; 25088 x 4096 -> 1024 with a residual 104 to 117 us, 1.8 to 2.0).
// O: the result's type; RES: a residual is added.  The result (and the residual) is whole runs (MatmulS8Args::out_runs).
template <typename O, bool RES, int MB>
__global__ __launch_bounds__(512, 2) void matmul_s8_walk_kernel(MatmulS8Args a, const int8_t* x, const int8_t* w, void* out)
{
    constexpr int WN = 4, WAVES = 8, BM = 32 * MB, BN = 256, BK = 128;
    constexpr int XL = (BM / 8 + WAVES - 1) / WAVES, WL = BN / 8 / WAVES;  // loads of a wave: 8 rows each
    constexpr int R = matmul_run(sizeof(O)), RUNS = 16 / R;
    __shared__ v4i lds[2 * (BM + BN) * 8];
    __shared__ float rows[BM], columns[2 * BN];  // of the tile that ends: scales of rows; scales of features, bias
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const v4i *xt = lds, *wt = lds + 2 * BM * 8;
    const uint32_t xl = lds_address(xt), wl = lds_address(wt);
    const int q = lane >> 4, r = lane & 15, wm = wave / WN, wn = wave - wm * WN;
    const int steps = (a.k + BK - 1) / BK, piece = (lane & 7) ^ (q | (wave & 1) << 2);
    const bool late = wave >= WAVES / 2;
    // the first of a run of a lane's values among the wave's 64 features
    const auto run = [&](int k) { return R == 4 ? 16 * k + 4 * q : 32 * k + 8 * q; };

    int m0, n0, xo[XL], wo[WL];
    v4i xs, ws;
    float row_value, column_value;
    const auto aim = [&](int tile) {
        int tm, tn, t = threadIdx.x;
        asm volatile("" : "+v"(t));  // (known, all of this would be worked out once for all tiles and kept in scratch memory)
        matmul_place(a, tile, tm, tn);
        m0 = tm * BM, n0 = tn * BN;
        xs = buffer_of(x + (int64_t)m0 * a.a_pitch), ws = buffer_of(w + (int64_t)n0 * a.w_pitch);
        const int of = (wave << 3) + (t >> 3 & 7);
#pragma unroll
        for (int i = 0; i < XL; ++i) xo[i] = min(i * WAVES * 8 + of, a.m - 1 - m0) * (int)a.a_pitch + 16 * piece;
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int row = i * WAVES * 8 + of, b = row & 63;
            const int feature = R == 4 ? b : (b & 32) + 8 * (b >> 2 & 3) + 4 * (b >> 4 & 1) + (b & 3);
            wo[i] = min((row & ~63) + feature, a.n - 1 - n0) * (int)a.w_pitch + 16 * piece;
        }
        row_value = 1.0f, column_value = t < BN ? 1.0f : 0.0f;
        if (a.a_scales && t < BM) row_value = a.a_scales[a.a_each ? min(m0 + t, a.m - 1) : 0];
        const int n = min(n0 + (t & (BN - 1)), a.n - 1);
        if (t < BN) {
            if (a.w_scales) column_value = a.w_scales[a.w_each ? n : 0];
        } else if (a.bias) column_value = a.bias[n];
    };
    const auto load = [&](int step, int at) {
        const int behind = step * BK + 16 * piece >= a.k ? (int)0x80000000 : 0;
#pragma unroll
        for (int i = 0; i < XL; ++i)
            if (BM / 8 % WAVES == 0 || i * WAVES + wave < BM / 8) load_lds(xs, xl + at * BM * 128 + (i * WAVES + wave) * 1024, xo[i] | behind, step * BK);
#pragma unroll
        for (int i = 0; i < WL; ++i) load_lds(ws, wl + at * BN * 128 + (i * WAVES + wave) * 1024, wo[i] | behind, step * BK);
    };
    v4i acc[4][MB], xf[MB], wf[4];
    const auto read = [&](int round, int at) {
        const int place = (4 * round + q) ^ (r >> 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) wf[j] = wt[at * BN * 8 + (wn * 64 + j * 16 + r) * 8 + place];
#pragma unroll
        for (int i = 0; i < MB; ++i) xf[i] = xt[at * BM * 8 + ((wm * MB + i) * 16 + r) * 8 + place];
    };
    const auto multiply = [&]() {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][i] = mfma16(wf[j], xf[i], acc[j][i]);
        __builtin_amdgcn_s_setprio(0);
    };
    int tile = blockIdx.x;
    aim(tile);
    load(0, 0);
    matmul_arrive<0>();
    for (;;) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][i] = v4i{0, 0, 0, 0};
        if (late) matmul_meet();
        for (int step = 0, at = 0; step < steps; ++step, at ^= 1) {
            load(step + 1, at ^ 1);
            read(0, at);
            matmul_meet();
            multiply();
            matmul_meet();
            read(1, at);
            // all reads of this buffer are done and the next step's loads have landed where the late waves end this phase
            if (late) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            matmul_meet();
            multiply();
            if (!late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            matmul_meet();
        }
        if (!late) matmul_meet();
        // nobody reads or fills the operands' LDS any more
        if (threadIdx.x < BM) rows[threadIdx.x] = row_value;
        columns[threadIdx.x] = column_value;
        const int m = m0 + wm * MB * 16, n = n0 + wn * 64;
        tile += gridDim.x;
        const bool more = tile < a.tiles;
        if (more) {
            aim(tile);
            load(0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

        float scale[16], bias[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int f = wn * 64 + (R == 4 ? run(g) : run(g >> 1) + 4 * (g & 1));
            const v4f s = *(const v4f*)&columns[f], b = *(const v4f*)&columns[BN + f];
#pragma unroll
            for (int l = 0; l < 4; ++l) scale[4 * g + l] = s[l], bias[4 * g + l] = b[l];
        }
        // Offsets from the wave's first value on.  Rows behind the last are behind the buffer's end, features behind the last are sent there.
        const auto buffer = [&](const void* base, int64_t pitch, int size) {
            const int64_t bytes = (a.m - m) * pitch * size;
            return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(base) + (m * pitch + n) * size, 0, m < a.m ? (int)min(bytes, (int64_t)0x7fffffff) : 0, 0x00020000);
        };
        const auto place = [&](int k, int64_t pitch, int size) { return n + run(k) < a.n ? r * (int)(pitch * size) + run(k) * size : (int)0x80000000; };
        const auto to = buffer(out, a.o_pitch, sizeof(O));
        int at[RUNS];
#pragma unroll
        for (int k = 0; k < RUNS; ++k) at[k] = place(k, a.o_pitch, sizeof(O));
        const int o_step = 16 * (int)(a.o_pitch * sizeof(O));
        const auto value = [&](int i, float (&v)[16]) {
            const float row = rows[(wm * MB + i) * 16 + r];
#pragma unroll
            for (int l = 0; l < 16; ++l) v[l] = __builtin_fmaf((float)acc[l / 4][i][l % 4] * row, scale[l], bias[l]);
        };
        const auto store = [&](int i, const float (&v)[16]) {
            typedef O vec __attribute__((ext_vector_type(R)));
#pragma unroll
            for (int k = 0; k < RUNS; ++k) {
                vec y;
#pragma unroll
                for (int l = 0; l < R; ++l) y[l] = (O)v[k * R + l];
                if (a.past) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, y), to, at[k] + i * o_step, 0, 2);
                else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, y), to, at[k] + i * o_step, 0, 0);
            }
        };
        if constexpr (RES) {
            const int size = a.res_type == CLDNN_HIP_F32 ? 4 : 2, r_step = 16 * (int)(a.r_pitch * size);
            const auto from = buffer(a.residual, a.r_pitch, size);
            int there[RUNS];
#pragma unroll
            for (int k = 0; k < RUNS; ++k) there[k] = place(k, a.r_pitch, size);
            const auto fetch = [&](int i) {
                v16u y{};
                const auto four = [&](int g, v4u z) { y[4 * g] = z[0], y[4 * g + 1] = z[1], y[4 * g + 2] = z[2], y[4 * g + 3] = z[3]; };
                if (size == 4) {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        four(g, __builtin_amdgcn_raw_buffer_load_b128(from, there[R == 4 ? g : g >> 1] + i * r_step + (R == 4 ? 0 : 16 * (g & 1)), 0, 0));
                } else if constexpr (R == 4) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const v2u z = __builtin_amdgcn_raw_buffer_load_b64(from, there[g] + i * r_step, 0, 0);
                        y[2 * g] = z[0], y[2 * g + 1] = z[1];
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < 2; ++g) four(g, __builtin_amdgcn_raw_buffer_load_b128(from, there[g] + i * r_step, 0, 0));
                }
                return y;
            };
            v16u now = fetch(0);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                v16u then{};
                if (i + 1 < MB) then = fetch(i + 1);
                float v[16];
                value(i, v);
                if (a.act.kind != CLDNN_HIP_ACT_NONE) act_apply<true>(v, a.act);
                matmul_typed(a.res_type, [&](auto t) { matmul_add_row<decltype(t)>(now, v); });
                if (a.act2.kind != CLDNN_HIP_ACT_NONE) act_apply<true>(v, a.act2);
                store(i, v);
                now = then;
            }
        } else {
            act_choose(a.act.kind, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    float v[16];
                    value(i, v);
#pragma unroll
                    for (int l = 0; l < 16; ++l) v[l] = act_one<decltype(kind)::value, true>(v[l], a.act.m, a.act.n);
                    store(i, v);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
        }
        if (!more) break;
        matmul_arrive<RUNS * MB>();  // the loads are older than the stores, of which there are so many
    }
}

namespace {

struct MatmulS8Kernel {
    const char* name;
    int rows, features, waves;
    int lds;  // bytes: the stages of both operands, or the waves' sums
    const char* walk;  // where the result is whole runs: the kernel that goes through several tiles, which has the scales in LDS besides
    int walk_lds() const { return lds + 4 * (rows + 2 * features); }
};
enum { MM_256, MM_224, MM_192, MM_128, MM_64x128, MM_64, MM_32, MM_ANY_64, MM_ANY_32, MM_16 };
const MatmulS8Kernel matmul_s8_kernels[] = {
    {"matmul_s8_tile<256x256>", 256, 256, 8, 128 << 10, "matmul_s8_walk<256x256>"}, {"matmul_s8_tile<224x256>", 224, 256, 8, 120 << 10, "matmul_s8_walk<224x256>"},
    {"matmul_s8_tile<192x256>", 192, 256, 8, 112 << 10, "matmul_s8_walk<192x256>"},
    {"matmul_s8_tile<128x128>", 128, 128, 4, 64 << 10}, {"matmul_s8_tile<64x128>", 64, 128, 4, 72 << 10},
    {"matmul_s8_tile<64x64,k2>", 64, 64, 8, 128 << 10}, {"matmul_s8_tile<32x64,k4>", 32, 64, 8, 144 << 10},
    {"matmul_s8_split<64x64>", 64, 64, 4, 64 << 10}, {"matmul_s8_split<32x32>", 32, 32, 8, 32 << 10}, {"matmul_s8_split<16x16>", 16, 16, 8, 8 << 10},
};

struct MatmulS8Plan : OperatorPlan {
    MatmulS8Args a{};
    int kernel = 0;  // row of matmul_s8_kernels; the one for any strides where pointers are not aligned
    int any = 0;
    int cus = 0;
    bool runs = false;  // sizes and strides allow whole runs of results
    int pieces = 0;  // > 0: the operands are copied into rows of so many 16-byte pieces first
};

int64_t pack_blocks(const MatmulS8Plan& p) { return (((int64_t)p.a.m + p.a.n) * p.pieces + MATMUL_PACK_THREADS - 1) / MATMUL_PACK_THREADS; }

int64_t count(int m, int n, const MatmulS8Kernel& k) { return (int64_t)((m + k.rows - 1) / k.rows) * ((n + k.features - 1) / k.features); }

// What a kernel takes in us behind a launch: for each round that its tiles need on the chip, base + step * K, measured over 324 sizes of 1 to
// 25088 rows, 96 to 8192 features and K of 256 to 16384 (f16 results).  Of two workgroups to a CU a full round has both, and a last
// one of at most one to a CU has the `one` figures.  The kernel with the least sum was the best at 315 of them and at most 7 % behind it
// at the others (profiles/operators_s8_kernel_choice.txt).
struct MatmulS8Time {
    int kernel, on_cu;  // workgroups to a CU
    double base, step, one_base, one_step;
};
const MatmulS8Time matmul_s8_times[] = {
    {MM_256, 1, 7.8, 0.0092}, {MM_224, 1, 7.0, 0.0086}, {MM_192, 1, 6.3, 0.0078}, {MM_128, 2, 6.0, 0.0062, 4.5, 0.0045},
    {MM_64x128, 2, 4.3, 0.0038, 3.9, 0.0027}, {MM_64, 1, 3.7, 0.0015}, {MM_32, 1, 3.7, 0.0011},
};

// whole: rows of 16-byte pieces, which the direct loads into LDS need
int choose(int m, int n, int k, bool whole, int cus)
{
    const auto tiles = [&](int row) { return count(m, n, matmul_s8_kernels[row]); };
    // Few tiles of any size: the smallest, whose eight waves split K.  (us, against 32 x 64 tiles: 32 x 256 -> 4096, 512 of them, 4.4 and 6.0,
    // 32 x 1024 -> 4096 5.3 and 6.5, 1 x 4096 -> 8192 8.6 and 10.5; every one reads all of its rows, so not many with a long K: 784 x 4096
    // -> 96, 294 of them, 10.5 and 9.0.  With more than 8 rows over a long K they are not more than the CUs where there is a choice: 16 x 8192
    // -> 5120, 320 of them, 17.7 and 13.5, 16 x 4096 -> 5120 10.7 and 9.4, 8 x 4096 -> 5120 9.4 and 9.3, 16 x 3008 -> 5120 7.4 and 8.4.)
    const int64_t few = tiles(MM_16);
    const bool heavy = whole && m > 8 && m <= 16 && k >= 4096;
    if (few <= (k <= 512 ? 3 * cus : heavy ? cus : k <= 1024 || m <= 16 ? 2 * cus : k <= 2048 || m <= 64 ? cus * 5 / 4 : cus)) return MM_16;
    if (!whole) return tiles(MM_ANY_64) >= cus ? MM_ANY_64 : MM_ANY_32;
    int best = MM_32;
    double least = 1e30;
    for (const MatmulS8Time& t : matmul_s8_times) {
        const int64_t all = tiles(t.kernel), full = all / (t.on_cu * cus), rest = all - full * t.on_cu * cus;
        const double round = t.base + t.step * k, last = t.on_cu > 1 && rest <= cus ? t.one_base + t.one_step * k : round;
        const double time = full * round + (rest ? last : 0.0);
        if (time < least) least = time, best = t.kernel;
    }
    return best;
}

void set_tiles(MatmulS8Args& a, const MatmulS8Kernel& k, const char* what)
{
    const int64_t tiles = count(a.m, a.n, k);
    check_grid(tiles, 64 * k.waves, what);
    a.tiles = (int32_t)tiles, a.tiles_m = (a.m + k.rows - 1) / k.rows, a.tiles_n = (a.n + k.features - 1) / k.features;
    a.band = 8;
}

}  // namespace

std::unique_ptr<OperatorPlan> matmul_s8_plan(const cldnn_hip_engine_s& e, const cldnn_hip_matmul_s8_desc& d, cldnn_hip_operator_info& info)
{
    CHIP_REQUIRE(d.m > 0 && d.n > 0 && d.k > 0, CLDNN_HIP_INVALID_ARG, "matmul s8: sizes must be positive");
    // so that a tile's last row or feature has a number
    CHIP_REQUIRE(std::max(d.m, d.n) <= INT32_MAX - 256, CLDNN_HIP_UNSUPPORTED_SIZE, "matmul s8: too large");
    CHIP_REQUIRE(d.k <= MATMUL_S8_MOST_K, CLDNN_HIP_UNSUPPORTED_SIZE, "matmul s8: k too large, more than 131071");
    const auto known = [](int scales) { return scales >= CLDNN_HIP_SCALES_NONE && scales <= CLDNN_HIP_SCALES_EACH; };
    CHIP_REQUIRE(known(d.a_scales) && known(d.weights_scales), CLDNN_HIP_INVALID_ARG, "matmul s8: unknown kind of scales");
    const int64_t out_size = float_size(d.out_dtype, "matmul s8");
    const int64_t res_size = d.residual_dtype == CLDNN_HIP_NO_TYPE ? 0 : float_size(d.residual_dtype, "matmul s8");
    CHIP_REQUIRE(res_size || d.residual_activation == CLDNN_HIP_ACT_NONE, CLDNN_HIP_INVALID_ARG, "matmul s8: an activation of the sum without a residual");
    std::unique_ptr<MatmulS8Plan> plan(new MatmulS8Plan());
    MatmulS8Args& a = plan->a;
    a.m = d.m, a.n = d.n, a.k = d.k;
    const auto pitch = [](int64_t stride, int64_t dense) {
        CHIP_REQUIRE(stride == 0 || stride >= dense, CLDNN_HIP_INVALID_ARG, "matmul s8: a stride shorter than its row");
        return stride ? stride : dense;
    };
    a.a_pitch = pitch(d.a_stride, d.k), a.w_pitch = pitch(d.weights_stride, d.k);
    a.o_pitch = pitch(d.out_stride, d.n), a.r_pitch = pitch(d.residual_stride, d.n);
    a.act = make_act(d.activation, d.activation_m, d.activation_n, "matmul s8");
    a.act2 = make_act(d.residual_activation, d.residual_activation_m, d.residual_activation_n, "matmul s8");
    a.out_type = d.out_dtype, a.res_type = d.residual_dtype;
    a.a_each = d.a_scales == CLDNN_HIP_SCALES_EACH, a.w_each = d.weights_scales == CLDNN_HIP_SCALES_EACH;
    // marks what the object has; enqueue puts the pointers there
    const auto mark = [](bool has) { return has ? (const float*)4 : nullptr; };
    a.a_scales = mark(d.a_scales != CLDNN_HIP_SCALES_NONE), a.w_scales = mark(d.weights_scales != CLDNN_HIP_SCALES_NONE);
    a.bias = mark(d.has_bias), a.residual = mark(res_size);
    const int run = matmul_run((int)out_size);
    const auto runs = [&](int64_t pitch) { return pitch % run == 0 && pitch <= MATMUL_S8_RUN_PITCH; };
    plan->runs = a.n % run == 0 && runs(a.o_pitch) && (!a.residual || runs(a.r_pitch));
    // A result of twice the dies' caches leaves them to the operands (us, through them and past them: behind a gelu 25088 x 1024 -> 4096, 196 MiB,
    // 138 and 130, 25088 x 512 -> 2048, 98 MiB, 57.1 and 53.5, 16384 x 1024 -> 2048, 64 MiB, 44.5 and 44.9; without one, in the same order, 122
    // and 118, 46.6 and 48.6, 40.8 and 46.9).  Half as large, a gelu's results gain 2 us of 24 to 38 and others lose as much (25088 x 1024 -> 1024,
    // 49 MiB, 38.5 and 37.4, 33.3 and 35.7).
    a.past = (int64_t)d.m * d.n * out_size >= MATMUL_S8_PAST;
    const int cus = plan->cus = e.props.multiProcessorCount;
    const bool whole = d.k % 16 == 0 && a.a_pitch % 16 == 0 && a.w_pitch % 16 == 0 && std::max(a.a_pitch, a.w_pitch) < (1 << 22);
    plan->kernel = choose(d.m, d.n, d.k, whole, cus);
    plan->any = choose(d.m, d.n, d.k, false, cus);
    if (!whole && plan->any != MM_16 && (double)d.m * d.n * d.k >= MATMUL_S8_PACK && ((int64_t)d.m + d.n) * ((d.k + 15) / 16) < (1ll << 32) - MATMUL_PACK_THREADS) {
        plan->pieces = (d.k + 15) / 16;
        plan->kernel = choose(d.m, d.n, d.k, true, cus);
    }
    const MatmulS8Kernel& kernel = matmul_s8_kernels[plan->kernel];
    set_tiles(a, kernel, "matmul s8");
    // The smallest tiles that leave half of the chip idle over a long K: workgroups that take 8192 of it each, a run of loads of their waves,
    // for the price of a second launch (us, one workgroup and several: 16 x 25088 -> 1000 24.9 and 13.8, 16 x 16384 -> 1000 17.0 and 13.1,
    // 1 x 16384 -> 500 11.6 and 9.9; 1 x 12288 -> 500 9.5 and 9.8; more and shorter parts gain nothing).
    a.splits = 1;
    if (plan->kernel == MM_16 && a.tiles * 2 <= cus && d.k > 12288) a.splits = std::min(cus / a.tiles, (d.k + 8191) / 8192);
    info.launches = plan->pieces || a.splits > 1 ? 2 : 1, info.block = 64 * kernel.waves, info.grid = a.tiles * a.splits, info.lds_bytes = kernel.lds;
    const bool walk = kernel.walk && plan->runs;
    if (walk) info.grid = std::min(a.tiles, cus), info.lds_bytes = kernel.walk_lds();
    if (plan->pieces) info.block = MATMUL_PACK_THREADS, info.grid = (int32_t)pack_blocks(*plan);
    info.workspace_bytes = ((int64_t)d.m + d.n) * plan->pieces * 16 + (a.splits > 1 ? (int64_t)a.splits * d.m * d.n * 4 : 0);
    info.ops = 2ll * d.m * d.n * d.k;
    const auto scales = [](int kind, int64_t rows) { return kind == CLDNN_HIP_SCALES_EACH ? 4 * rows : kind == CLDNN_HIP_SCALES_ONE ? 4 : 0; };
    info.bytes = (int64_t)d.m * d.k + (int64_t)d.n * d.k + scales(d.a_scales, d.m) + scales(d.weights_scales, d.n) + (d.has_bias ? 4ll * d.n : 0) +
                 (int64_t)d.m * d.n * (out_size + res_size);
    snprintf(info.kernel_name, sizeof info.kernel_name, "%s%s%s", plan->pieces ? "matmul_pack + " : "", walk ? kernel.walk : kernel.name, a.splits > 1 ? " + matmul_join" : "");
    return plan;
}

void matmul_s8_launch(hipStream_t s, const OperatorPlan& plan, void* workspace, const void* x, const void* w, const float* a_scales, const float* w_scales, const float* bias,
                      const void* residual, void* out)
{
    const MatmulS8Plan& p = static_cast<const MatmulS8Plan&>(plan);
    MatmulS8Args a = p.a;
    CHIP_REQUIRE((!a.bias || bias) && (!a.residual || residual) && (!a.a_scales || a_scales) && (!a.w_scales || w_scales), CLDNN_HIP_INVALID_ARG, "null device pointer");
    check_aligned(out, float_size(a.out_type, ""), "output");
    if (a.a_scales) check_aligned(a_scales, 4, "a_scales"), a.a_scales = a_scales;
    if (a.w_scales) check_aligned(w_scales, 4, "weights_scales"), a.w_scales = w_scales;
    if (a.bias) check_aligned(bias, 4, "bias"), a.bias = bias;
    if (a.residual) check_aligned(residual, float_size(a.res_type, ""), "residual"), a.residual = residual;
    const auto whole = [&](const void* p, int type) { return ((uintptr_t)p & (std::min(16, matmul_run(float_size(a.out_type, "")) * float_size(type, "")) - 1)) == 0; };
    a.out_runs = p.runs && whole(out, a.out_type) && (!a.residual || whole(residual, a.res_type));
    const int8_t *xa = (const int8_t*)x, *wa = (const int8_t*)w;
    a.part = workspace;
    if (p.pieces) {
        hipLaunchKernelGGL((matmul_pack_kernel<int8_t>), dim3((unsigned)pack_blocks(p)), dim3(MATMUL_PACK_THREADS), 0, s, a, xa, wa, (v4i*)workspace, p.pieces);
        a.a_pitch = a.w_pitch = a.k = 16 * p.pieces;
        xa = (const int8_t*)workspace, wa = xa + (int64_t)a.m * a.a_pitch;
    }
    const int row = (((uintptr_t)xa | (uintptr_t)wa) & 15) == 0 ? p.kernel : p.any;
    const MatmulS8Kernel& kernel = matmul_s8_kernels[row];
    set_tiles(a, kernel, row == p.kernel ? "matmul s8" : "matmul s8, operands that are not aligned to 16 bytes");
    const auto launch = [&](auto f) { hipLaunchKernelGGL(f, dim3(kernel.walk && a.out_runs ? std::min(a.tiles, p.cus) : a.tiles, a.splits), dim3(64 * kernel.waves), 0, s, a, xa, wa, out); };
    const auto large = [&](auto mb) {
        constexpr int MB = decltype(mb)::value;
        if (!a.out_runs) return launch(matmul_tile_kernel<int8_t, 2, 4, MB, 2, 1>);
        with_float(a.out_type, [&](auto o) { launch(a.residual ? matmul_s8_walk_kernel<decltype(o), true, MB> : matmul_s8_walk_kernel<decltype(o), false, MB>); });
    };
    switch (row) {
    case MM_256: large(std::integral_constant<int, 8>()); break;
    case MM_224: large(std::integral_constant<int, 7>()); break;
    case MM_192: large(std::integral_constant<int, 6>()); break;
    case MM_128: launch(matmul_tile_kernel<int8_t, 2, 2, 4, 2, 1>); break;
    case MM_64x128: launch(matmul_tile_kernel<int8_t, 2, 2, 2, 3, 1>); break;
    case MM_64: launch(matmul_tile_kernel<int8_t, 4, 1, 1, 4, 2>); break;
    case MM_32: launch(matmul_tile_kernel<int8_t, 2, 1, 1, 3, 4>); break;
    case MM_ANY_64: launch(matmul_split_kernel<int8_t, 4, 4, 2, 4>); break;
    case MM_ANY_32: launch(matmul_split_kernel<int8_t, 2, 2, 4, 8>); break;
    default: launch(matmul_split_kernel<int8_t, 1, 1, 16, 8>);
    }
    if (a.splits > 1)
        hipLaunchKernelGGL((matmul_join_kernel<int8_t>), dim3((unsigned)(((int64_t)a.m * ((a.n + 3) / 4) + 255) / 256)), dim3(256), 0, s, a, out);
    CHIP_CHECK(hipGetLastError());
}

}  // namespace chip
