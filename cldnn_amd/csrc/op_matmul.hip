// Matrix product with bias, activation and residual: out = act2(act(a w^T + bias) + residual).
#include "matmul_kernel.h"

namespace chip {

constexpr int64_t MATMUL_PACK = 200ll << 20;  // products from which unaligned operands are copied

struct MatmulPlan {
    MatmulFloatArgs a;
    int dt;
    int kernel;  // row of matmul_kernels; the one for any strides where pointers are not aligned
    int any;
    int pieces;  // > 0: the operands are copied into rows of so many 16-byte pieces first
};


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
    MatmulFloatArgs& a = plan->a;
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
    MatmulFloatArgs a = p.a;
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
