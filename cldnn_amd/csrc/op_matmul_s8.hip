// Matrix product of int8 operands with scales for each row and channel: out = act2(act(a w^T * row * channel + bias) + residual).
// The kernels are those of the float products (matmul_kernel.h): a row of either type is the same pieces of 16 bytes.
#include "matmul_kernel.h"
#include "ops_s8.h"

namespace chip {

constexpr int MATMUL_S8_MOST_K = 131071;  // 128 * 128 of each fit 31 bits
constexpr int64_t MATMUL_S8_PACK = 200ll << 20;  // products from which unaligned operands are copied

namespace {

struct MatmulS8Kernel {
    const char* name;
    int rows, features, waves;
    int lds;  // bytes: the stages of both operands, or the waves' sums
};
enum { MM_256, MM_224, MM_192, MM_128, MM_64x128, MM_64, MM_32, MM_ANY_64, MM_ANY_32, MM_16 };
const MatmulS8Kernel matmul_s8_kernels[] = {
    {"matmul_s8_tile<256x256>", 256, 256, 8, 128 << 10}, {"matmul_s8_tile<224x256>", 224, 256, 8, 120 << 10}, {"matmul_s8_tile<192x256>", 192, 256, 8, 112 << 10},
    {"matmul_s8_tile<128x128>", 128, 128, 4, 64 << 10}, {"matmul_s8_tile<64x128>", 64, 128, 4, 72 << 10},
    {"matmul_s8_tile<64x64,k2>", 64, 64, 8, 128 << 10}, {"matmul_s8_tile<32x64,k4>", 32, 64, 8, 144 << 10},
    {"matmul_s8_split<64x64>", 64, 64, 4, 64 << 10}, {"matmul_s8_split<32x32>", 32, 32, 8, 32 << 10}, {"matmul_s8_split<16x16>", 16, 16, 8, 8 << 10},
};

struct MatmulS8Plan : OperatorPlan {
    MatmulS8Args a{};
    int kernel = 0;  // row of matmul_s8_kernels; the one for any strides where pointers are not aligned
    int any = 0;
    int pieces = 0;  // > 0: the operands are copied into rows of so many 16-byte pieces first
};

int64_t pack_blocks(const MatmulS8Plan& p) { return (((int64_t)p.a.m + p.a.n) * p.pieces + MATMUL_PACK_THREADS - 1) / MATMUL_PACK_THREADS; }

int64_t count(int m, int n, const MatmulS8Kernel& k) { return (int64_t)((m + k.rows - 1) / k.rows) * ((n + k.features - 1) / k.features); }

// whole: rows of 16-byte pieces, which the direct loads into LDS need
int choose(int m, int n, bool whole, int cus)
{
    const auto tiles = [&](int row) { return count(m, n, matmul_s8_kernels[row]); };
    const auto rounds = [&](int row) { return (tiles(row) + cus - 1) / cus; };
    if (tiles(MM_16) * 4 <= cus * 5) return MM_16;
    if (!whole) return tiles(MM_ANY_64) >= cus ? MM_ANY_64 : MM_ANY_32;
    if (tiles(MM_128) * 4 >= cus * 5) {
        const int kernel[] = {MM_256, MM_224, MM_192, MM_128};
        const double time[] = {rounds(MM_256) * 256.0, rounds(MM_224) * 224 * 1.04, rounds(MM_192) * 192 * 1.12, rounds(MM_128) * 64 * 1.22};
        return kernel[std::min_element(time, time + 4) - time];
    }
    if (tiles(MM_64x128) * 4 >= cus * 3) return MM_64x128;
    if (tiles(MM_64) * 4 >= cus * 3) return MM_64;
    return MM_32;
}

void set_tiles(MatmulS8Args& a, const MatmulS8Kernel& k)
{
    const int64_t tiles = count(a.m, a.n, k);
    check_grid(tiles, 64 * k.waves, "matmul s8");
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
    const int cus = e.props.multiProcessorCount;
    const bool whole = d.k % 16 == 0 && a.a_pitch % 16 == 0 && a.w_pitch % 16 == 0 && std::max(a.a_pitch, a.w_pitch) < (1 << 22);
    plan->kernel = choose(d.m, d.n, whole, cus);
    plan->any = choose(d.m, d.n, false, cus);
    if (!whole && plan->any != MM_16 && (double)d.m * d.n * d.k >= MATMUL_S8_PACK && ((int64_t)d.m + d.n) * ((d.k + 15) / 16) < (1ll << 32) - MATMUL_PACK_THREADS) {
        plan->pieces = (d.k + 15) / 16;
        plan->kernel = choose(d.m, d.n, true, cus);
    }
    const MatmulS8Kernel& kernel = matmul_s8_kernels[plan->kernel];
    set_tiles(a, kernel);
    a.splits = 1;
    if (plan->kernel == MM_16 && a.tiles * 2 <= cus && d.k >= 16000) a.splits = std::min(cus / a.tiles, d.k / 4096);
    info.launches = plan->pieces || a.splits > 1 ? 2 : 1, info.block = 64 * kernel.waves, info.grid = a.tiles * a.splits, info.lds_bytes = kernel.lds;
    if (plan->pieces) info.block = MATMUL_PACK_THREADS, info.grid = (int32_t)pack_blocks(*plan);
    info.workspace_bytes = ((int64_t)d.m + d.n) * plan->pieces * 16 + (a.splits > 1 ? (int64_t)a.splits * d.m * d.n * 4 : 0);
    info.ops = 2ll * d.m * d.n * d.k;
    const auto scales = [](int kind, int64_t rows) { return kind == CLDNN_HIP_SCALES_EACH ? 4 * rows : kind == CLDNN_HIP_SCALES_ONE ? 4 : 0; };
    info.bytes = (int64_t)d.m * d.k + (int64_t)d.n * d.k + scales(d.a_scales, d.m) + scales(d.weights_scales, d.n) + (d.has_bias ? 4ll * d.n : 0) +
                 (int64_t)d.m * d.n * (out_size + res_size);
    snprintf(info.kernel_name, sizeof info.kernel_name, "%s%s%s", plan->pieces ? "matmul_pack + " : "", kernel.name, a.splits > 1 ? " + matmul_join" : "");
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
    const int8_t *xa = (const int8_t*)x, *wa = (const int8_t*)w;
    a.part = workspace;
    if (p.pieces) {
        hipLaunchKernelGGL((matmul_pack_kernel<int8_t>), dim3((unsigned)pack_blocks(p)), dim3(MATMUL_PACK_THREADS), 0, s, a, xa, wa, (v4i*)workspace, p.pieces);
        a.a_pitch = a.w_pitch = a.k = 16 * p.pieces;
        xa = (const int8_t*)workspace, wa = xa + (int64_t)a.m * a.a_pitch;
    }
    const int row = (((uintptr_t)xa | (uintptr_t)wa) & 15) == 0 ? p.kernel : p.any;
    const MatmulS8Kernel& kernel = matmul_s8_kernels[row];
    set_tiles(a, kernel);
    const auto launch = [&](auto f) { hipLaunchKernelGGL(f, dim3(a.tiles, a.splits), dim3(64 * kernel.waves), 0, s, a, xa, wa, out); };
    switch (row) {
    case MM_256: launch(matmul_tile_kernel<int8_t, 2, 4, 8, 2, 1>); break;
    case MM_224: launch(matmul_tile_kernel<int8_t, 2, 4, 7, 2, 1>); break;
    case MM_192: launch(matmul_tile_kernel<int8_t, 2, 4, 6, 2, 1>); break;
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
