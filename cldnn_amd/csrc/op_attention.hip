// Attention in one pass over the keys with the running maximum and sum of the softmax.
//
// A wave has 32 rows: the queries of one key head, those of its sharing heads side by side.  It computes the scores transposed,
// S^T = K Q^T, so that a row of the softmax lies in the registers of two lanes (32 apart), and the result transposed as well,
// O^T = V^T P^T: the registers that S^T leaves in a lane are, as they lie, the operand that this second product wants, provided
// that V's keys are taken in the same order: in a step of 16 keys lane half h has keys 4h..4h+3 and 8+4h..8+4h+3.  That is what
// the transposing LDS read gives, four keys of a value to a lane.
// Values 16h + 4i + c of a block of 32 are put into row 8i + 4h + c of V^T, so a lane ends with 16 neighbouring values of its row.
//
// Measured (bf16, batch 4, 8 heads): 4096 x 4096 of 64 146 us (0.94 PFLOP/s), of 128 267 us (1.03); 3136 x 3136 of 64 105 us, where the
// fullest CUs have two workgroups and the mean is 1.6.  The vector units are busy in two thirds of the time (32 exponentials at 8
// clocks and 100 other instructions a tile and wave, 790 clocks), the matrix units in 43 % (512 clocks), at the 1.9 GHz that the power
// limit leaves.  Scores of the next tile under the exponentials of this one were no faster (three waves to a SIMD instead of four).
// One query over 50176 keys of 2 x 2 heads of 128: 24 us for lengths of 3/4 on average, 19 of it the keys at 4 TB/s.
//
// The probabilities are rounded to the data's type, the one that the second product takes them in; sums, maxima and results are not.
// It takes the result from 0.0017 to 0.0023 of its size away from the formula in 64 bits (bf16, 3136 x 3136 of 64; f16, 49 x 49: 0.00021
// and 0.00025; the first is what the result's own rounding makes).  The products of the probability and of what its rounding left,
// added up, would come as near as that, for half as many matrix instructions again.
//
// The waves of a workgroup share tiles of 64 keys, which direct loads bring into LDS one tile ahead.  Where rows are few the keys
// are split over workgroups (of one wave then), and a second kernel joins their parts.
#include <cfloat>

#include "ops_common.h"

namespace chip {

struct AttentionArgs {
    int32_t q_len, kv_len, kv_heads, group, head, rows;  // rows = q_len * group
    int32_t blocks, splits, total;                       // workgroups along the rows, along the keys, in all
    int32_t negative;                                    // scale < 0: the queries change their sign
    float scale;   // of the scores, with a bias only: without one they stay as the product leaves them
    float unit;    // of a score in powers of two.  With a bias log2(e): there a bias of the lowest value has to stay finite
    float margin;  // 8 powers of two
    int64_t q_pb, q_pt, q_ph, k_pb, k_pt, k_ph, v_pb, v_pt, v_ph, o_pb, o_pt, o_ph, b_pb, b_ph, b_pq;
};

struct AttentionPlan {
    AttentionArgs a;
    int dt, batch, size, bias_dt, has_lengths;
    int waves;
    int far;  // keys too far apart for 32-bit offsets within a tile
};

constexpr int ATT_KEYS = 64;  // of a tile
constexpr float ATT_LARGE = 4096.0f;  // powers of two from which on a score's product with its unit is not good to 12 bits behind the point
constexpr int ATT_ONE_WAVE = 128;  // largest head that a workgroup of one wave is made for: beyond, a CU holds one tile anyway

// Piece c (16 bytes) of row r of D values lies at place r * D / 8 + (c ^ att_turn(r)) of a tile in LDS: sixteen neighbouring rows
// have a piece in all 64 banks, and so have four rows four neighbouring pieces, which the transposing read takes at a time.
template <int D>
__device__ inline int att_turn(int r)
{
    if constexpr (D % 128 == 0) return (r & 1) << 3 | (r & 2) << 1 | (r >> 1 & 2) | (r >> 3 & 1);
    if constexpr (D % 64 == 0) return (r << 1 & 4) | (r >> 1 & 2) | (r >> 3 & 1);
    return r >> 2 & 3;
}

template <typename T>
__device__ inline v2i att_read_turned(const v4i* tile, int at)
{
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s* ptr;
    return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)((const __attribute__((address_space(3))) char*)tile + at)));
}

// The largest of three.  Written out: fmaxf turns signalling NaNs of its operands quiet first, an instruction for each score.  `a`
// has to depend on an ordinary instruction that read the last of the matrix instructions that b and c come from: the compiler
// counts the wait states of their results for that one.
__device__ inline float att_max(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// f of a lane's value and that of the lane 32 apart
template <typename F>
__device__ inline float att_both(float x, F&& f)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return f(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// sum + a + b in one instruction, of probabilities as they are rounded: bf16 only, whose smallest values no sum misses
__device__ inline float att_add(__bf16 a, __bf16 b, float sum)
{
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(v2b{a, b}, v2b{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
}
__device__ inline float att_add(_Float16 a, _Float16 b, float sum) { return sum + (float)a + (float)b; }

// Waves to a SIMD: what the registers of four and eight waves sharing a tile leave.  A workgroup of one wave has a tile of its own, and
// LDS holds two to ten of those to a CU (D 128 to 32).  Of all, heads up to 160 with an f32 bias and up to 256 with keys that are far
// apart and a bias run out of registers, by 3 to 26 that lie in scratch memory.
template <typename T, int D, typename B, int WAVES, bool FAR>
__global__ __launch_bounds__(64 * WAVES, WAVES == 1 ? (D <= 32 ? 3 : 1) : D <= 64 ? (std::is_same<B, void>::value ? 4 : 3) : D <= 160 ? 2 : 1) void attention_kernel(AttentionArgs a, const T* q, const T* k, const T* v, const int32_t* lengths, const B* bias, T* out, float* part)
{
    typedef typename vec8<T>::type V8;
    constexpr int C = D / 8, STEPS = D / 16, BLOCKS = D / 32, TILE = ATT_KEYS * C, LOADS = C / WAVES;
    constexpr bool BIAS = !std::is_same<B, void>::value, ROUNDED = std::is_same<T, __bf16>::value;
    __shared__ v4i kt[2 * TILE], vt[2 * TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    // as in the matrix product each die gets a run of workgroups: those of one head share its keys there
    const int die = blockIdx.x & 7;
    int block = die * (a.total >> 3) + min(die, a.total & 7) + (blockIdx.x >> 3);
    const int pair_split = block / a.blocks;
    block -= pair_split * a.blocks;
    const int pair = pair_split / a.splits, split = pair_split - pair * a.splits, b = pair / a.kv_heads, kh = pair - b * a.kv_heads;
    const int own = (block * WAVES + wave) * 32 + col, row = min(own, a.rows - 1);
    const int qi = row / a.group, h = kh * a.group + row - qi * a.group;
    const int length = lengths ? min(max(lengths[b], 0), a.kv_len) : a.kv_len;
    const int tiles = (length + ATT_KEYS - 1) / ATT_KEYS;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int chunks = a.head / 8;

    V8 qf[STEPS];
    const T* qr = q + b * a.q_pb + qi * a.q_pt + h * a.q_ph;
    const int sign = a.negative ? (int)0x80008000 : 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int c = 2 * s + half;
        v4i x = {0, 0, 0, 0};
        if (c < chunks) x = *(const v4i*)(qr + 8 * c) ^ v4i{sign, sign, sign, sign};
        qf[s] = __builtin_bit_cast(V8, x);
    }
    const T* kb = k + b * a.k_pb + kh * a.k_ph;
    const T* vb = v + b * a.v_pb + kh * a.v_ph;

    // the tile's rows from a length on and the pieces behind the head are zeros
    int ko[LOADS], vo[LOADS], key_of[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = (i * WAVES + wave) * 64 + lane, key = at / C, c = (at - key * C) ^ att_turn<D>(key);
        key_of[i] = c < chunks ? key : 1 << 30;
        if constexpr (!FAR) ko[i] = key * (int)(a.k_pt * 2) + 16 * c, vo[i] = key * (int)(a.v_pt * 2) + 16 * c;
    }
    const auto load = [&](int tile, int at) {
        const int key0 = tile * ATT_KEYS;
        if constexpr (FAR) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int to = (i * WAVES + wave) * 64 + lane, key = to / C, c = (to - key * C) ^ att_turn<D>(key);
                const bool there = key_of[i] < length - key0;
                kt[at * TILE + to] = there ? *(const v4i*)(kb + (int64_t)(key0 + key) * a.k_pt + 8 * c) : v4i{0, 0, 0, 0};
                vt[at * TILE + to] = there ? *(const v4i*)(vb + (int64_t)(key0 + key) * a.v_pt + 8 * c) : v4i{0, 0, 0, 0};
            }
        } else {
            const v4i ks = buffer_of(kb + (int64_t)key0 * a.k_pt), vs = buffer_of(vb + (int64_t)key0 * a.v_pt);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int behind = key_of[i] < length - key0 ? 0 : (int)0x80000000;
                load_lds(ks, lds_address(kt) + at * TILE * 16 + (i * WAVES + wave) * 1024, ko[i] | behind, 0);
                load_lds(vs, lds_address(vt) + at * TILE * 16 + (i * WAVES + wave) * 1024, vo[i] | behind, 0);
            }
        }
    };

    // where the lane reads V: key 4 half + lane / 4 % 4 (+ 8) of a step, four values from 16 h + 4 i on
    int vp[2][BLOCKS];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) {
            const int r = 8 * j + 4 * half + (lane >> 2 & 3), quad = (lane >> 4 & 1) * 4 + (lane & 3);
            const int d = 32 * i + 16 * (quad & 1) + 4 * (quad >> 1);
            vp[j][i] = (r * C + ((d / 8) ^ att_turn<D>(r))) * 16 + (d & 4) * 2;
        }

    v16f o[BLOCKS] = {};
    float most = -INFINITY, sum = 0.0f;
    float base = 0.0f, under = 0.0f;  // the maximum, and its product with the unit, that the exponents are taken from
    bool large = false;
    if (first < last) load(first, 0);
    for (int tile = first, at = 0; tile < last; ++tile, at ^= 1) {
        if constexpr (FAR) __syncthreads();
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (tile + 1 < last) load(tile + 1, at ^ 1);
        const v4i* kl = kt + at * TILE;
        v16f s[2] = {};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                s[t] = mfma32(__builtin_bit_cast(V8, kl[(32 * t + col) * C + ((2 * i + half) ^ att_turn<D>(col))]), qf[i], s[t]);
        __builtin_amdgcn_s_setprio(0);
        const int key0 = tile * ATT_KEYS;
        if constexpr (BIAS) {
            const B* at_bias = bias + b * a.b_pb + h * a.b_ph + qi * a.b_pq;
            typedef B any __attribute__((ext_vector_type(4), aligned(sizeof(B))));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 32 * t + 8 * i + 4 * half;
                    any x = {};
                    if (key + 4 <= a.kv_len) x = *(const any*)(at_bias + key);
                    else
                        for (int j = 0; j < 3; ++j)
                            if (key + j < a.kv_len) x[j] = at_bias[key + j];
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[t][4 * i + j] = __builtin_fmaf(s[t][4 * i + j], a.scale, (float)x[j]);
                }
        }
        if (key0 + ATT_KEYS > length)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + 32 * t + 8 * (i / 4) + 4 * half + i % 4 >= length) s[t][i] = -INFINITY;
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) top = att_max(top, s[0][i], s[1][i]);
        top = att_both(top, [](float x, float y) { return fmaxf(x, y); });
        // The maximum that the exponents are taken from follows when it is left behind by 2^8, which the sums and the operands of the
        // second product hold without loss: after the first tiles hardly ever.
        if (__any(top > most + a.margin) || large) {
            const bool follow = top > most + a.margin;
            const float fade = follow ? __builtin_amdgcn_exp2f((most - top) * a.unit) : 1.0f;
            most = follow ? top : most;
            sum *= fade;
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= fade;
            base = most == -INFINITY ? 0.0f : most;  // a row without a key so far
            if constexpr (!BIAS) {
                // The rounding of a large product with the unit would show in the exponents, where it no longer is that of the scores
                // alone: they are taken from the maximum first then.
                under = base * a.unit;
                large = __any(__builtin_fabsf(under) > ATT_LARGE);
                if (large) {
                    under = 0.0f;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[t][i] -= base;
                }
            }
        }
        V8 p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(BIAS ? (s[t][i] - base) * a.unit : __builtin_fmaf(s[t][i], a.unit, -under));
                if constexpr (!ROUNDED) sum += e;
                p[2 * t + i / 8][i % 8] = (T)e;
            }
        if constexpr (ROUNDED)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; j += 2) sum = att_add(p[i][j], p[i][j + 1], sum);
        const v4i* vl = vt + at * TILE;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
                const v2i lo = att_read_turned<T>(vl, vp[0][i] + st * 16 * C * 16), hi = att_read_turned<T>(vl, vp[1][i] + st * 16 * C * 16);
                o[i] = mfma32(__builtin_bit_cast(V8, v4i{lo[0], lo[1], hi[0], hi[1]}), p[st], o[i]);
            }
        __builtin_amdgcn_s_setprio(0);
    }
    sum = att_both(sum, [](float x, float y) { return x + y; });
    if (own >= a.rows) return;
    if (a.splits > 1) {
        const int64_t at = (int64_t)pair_split * a.rows + row;
        float* to = part + at * a.head;
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 32 * i + 16 * half + 4 * j;
                if (d < a.head) *(v4f*)(to + d) = v4f{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
            }
        float2* ends = (float2*)(part + (int64_t)(a.total / a.blocks) * a.rows * a.head);
        if (half == 0) ends[at] = make_float2(most, sum);
        return;
    }
    const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* to = out + b * a.o_pb + qi * a.o_pt + h * a.o_ph;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int d = 32 * i + 16 * half + 8 * j;
            V8 x;
#pragma unroll
            for (int l = 0; l < 8; ++l) x[l] = (T)(o[i][8 * j + l] * factor);
            if (d < a.head) *(V8*)(to + d) = x;
        }
}

// Joins the parts of a row: each is moved to the largest of their maxima.  One workgroup to a row of a head pair; four values to a
// thread, so that few rounds of loads lie one behind the other (128 parts of a row of 128: 18 us with a value and 2 parts at a time).
constexpr int ATT_JOIN = 512, ATT_MOST_SPLITS = 1024;
template <typename T>
__global__ __launch_bounds__(ATT_JOIN) void attention_join_kernel(AttentionArgs a, const float* part, T* out)
{
    __shared__ float weight[ATT_MOST_SPLITS], both[2][ATT_JOIN / 64];
    __shared__ v4f values[ATT_JOIN];
    const int row = blockIdx.x, pair = blockIdx.y, b = pair / a.kv_heads, kh = pair - b * a.kv_heads, t = threadIdx.x;
    const int64_t at0 = (int64_t)pair * a.splits * a.rows + row;
    const float2* ends = (const float2*)(part + (int64_t)(a.total / a.blocks) * a.rows * a.head);
    // the parts' values are asked for before their weights are known
    const int lanes = a.head / 4, turns = ATT_JOIN / lanes, turn = t / lanes, d = (t - turn * lanes) * 4;
    const bool live = turn < turns;
    const auto value = [&](int s) { return live && s < a.splits ? *(const v4f*)(part + (at0 + (int64_t)s * a.rows) * a.head + d) : v4f{0, 0, 0, 0}; };
    v4f first[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) first[i] = value(turn + i * turns);
    float2 end[ATT_MOST_SPLITS / ATT_JOIN];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < ATT_MOST_SPLITS / ATT_JOIN; ++i) {
        const int s = t + i * ATT_JOIN;
        end[i] = s < a.splits ? ends[at0 + (int64_t)s * a.rows] : make_float2(-INFINITY, 0.0f);
        most = fmaxf(most, end[i].x);
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) most = fmaxf(most, __shfl_xor(most, i));
    if ((t & 63) == 0) both[0][t >> 6] = most;
    __syncthreads();
    for (int i = 0; i < ATT_JOIN / 64; ++i) most = fmaxf(most, both[0][i]);
    if (most == -INFINITY) most = 0.0f;  // no key in any part
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ATT_MOST_SPLITS / ATT_JOIN; ++i) {
        const float w = __builtin_amdgcn_exp2f((end[i].x - most) * a.unit);
        if (t + i * ATT_JOIN < a.splits) weight[t + i * ATT_JOIN] = w;
        sum = __builtin_fmaf(w, end[i].y, sum);
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    if ((t & 63) == 0) both[1][t >> 6] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int i = 0; i < ATT_JOIN / 64; ++i) sum += both[1][i];
    v4f v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (live && turn + i * turns < a.splits) v += first[i] * weight[turn + i * turns];
    for (int s = turn + 4 * turns; live && s < a.splits; s += turns) v += value(s) * weight[s];
    values[t] = v;
    __syncthreads();
    if (t >= a.head) return;
    float x = 0.0f;
    for (int i = 0; i < turns; ++i) x += ((const float*)values)[i * a.head + t];
    const int qi = row / a.group, h = kh * a.group + row - qi * a.group;
    out[b * a.o_pb + qi * a.o_pt + h * a.o_ph + t] = (T)(sum == 0.0f ? 0.0f : x / sum);
}

AttentionPlan* attention_plan(const cldnn_hip_engine_s& e, const cldnn_hip_attention_desc& d, cldnn_hip_operator_info& info)
{
    const auto is_half = [](int dt) { return dt == CLDNN_HIP_F16 || dt == CLDNN_HIP_BF16; };
    CHIP_REQUIRE(d.batch > 0 && d.q_len > 0 && d.kv_len > 0 && d.q_heads > 0 && d.kv_heads > 0 && d.head_size > 0, CLDNN_HIP_INVALID_ARG,
                 "attention: sizes must be positive");
    CHIP_REQUIRE(d.q_heads % d.kv_heads == 0, CLDNN_HIP_DIMENSION_MISMATCH, "attention: the key heads must divide the query heads");
    CHIP_REQUIRE(is_half(d.dtype), CLDNN_HIP_INVALID_ARG, "attention: data must be f16 or bf16");
    CHIP_REQUIRE(d.bias_dtype == d.dtype || d.bias_dtype == CLDNN_HIP_F32 || d.bias_dtype == CLDNN_HIP_NO_TYPE, CLDNN_HIP_INVALID_ARG,
                 "attention: the bias must be of the data's type or f32");
    CHIP_REQUIRE(d.head_size % 8 == 0 && d.head_size <= 256, CLDNN_HIP_UNSUPPORTED_SIZE, "attention: head_size must be a multiple of 8 up to 256");
    CHIP_REQUIRE(d.scale == d.scale && d.scale - d.scale == 0.0f, CLDNN_HIP_INVALID_ARG, "attention: the scale must be finite");
    std::unique_ptr<AttentionPlan> plan(new AttentionPlan{});
    AttentionArgs& a = plan->a;
    a.q_len = d.q_len, a.kv_len = d.kv_len, a.kv_heads = d.kv_heads, a.group = d.q_heads / d.kv_heads, a.head = d.head_size;
    const int64_t rows = (int64_t)d.q_len * a.group;
    CHIP_REQUIRE(rows < (1ll << 31) - 256 && d.batch <= 65535 && d.kv_heads <= 65535 && d.kv_len < (1 << 30), CLDNN_HIP_UNSUPPORTED_SIZE, "attention: too large");
    a.rows = (int32_t)rows;
    const float scale = d.scale != 0.0f ? d.scale : 1.0f / std::sqrt((float)d.head_size);
    a.negative = scale < 0.0f;
    a.scale = std::fabs(scale);
    a.unit = 1.44269504f * (d.bias_dtype == CLDNN_HIP_NO_TYPE ? a.scale : 1.0f);
    CHIP_REQUIRE(std::isfinite(a.unit), CLDNN_HIP_INVALID_ARG, "attention: a scale too large for 32 bits");
    a.margin = std::min(8.0f / a.unit, FLT_MAX);  // minus infinity stays below every score
    const auto strides = [&](int heads, int len, int64_t batch, int64_t token, int64_t head, int64_t& pb, int64_t& pt, int64_t& ph) {
        ph = head ? head : d.head_size;
        pt = token ? token : (int64_t)heads * d.head_size;
        pb = batch ? batch : pt * len;
        CHIP_REQUIRE(pb > 0 && pt > 0 && ph > 0, CLDNN_HIP_INVALID_ARG, "attention: strides must not be negative");
        CHIP_REQUIRE(pb % 8 == 0 && pt % 8 == 0 && ph % 8 == 0, CLDNN_HIP_UNSUPPORTED_FORMAT, "attention: strides must be multiples of 8 elements");
    };
    strides(d.q_heads, d.q_len, d.q_batch_stride, d.q_token_stride, d.q_head_stride, a.q_pb, a.q_pt, a.q_ph);
    strides(d.kv_heads, d.kv_len, d.k_batch_stride, d.k_token_stride, d.k_head_stride, a.k_pb, a.k_pt, a.k_ph);
    strides(d.kv_heads, d.kv_len, d.v_batch_stride, d.v_token_stride, d.v_head_stride, a.v_pb, a.v_pt, a.v_ph);
    strides(d.q_heads, d.q_len, d.out_batch_stride, d.out_token_stride, d.out_head_stride, a.o_pb, a.o_pt, a.o_ph);
    CHIP_REQUIRE(d.bias_batch_stride >= 0 && d.bias_head_stride >= 0 && d.bias_q_stride >= 0, CLDNN_HIP_INVALID_ARG, "attention: strides must not be negative");
    a.b_pb = d.bias_batch_stride, a.b_ph = d.bias_head_stride, a.b_pq = d.bias_q_stride;
    plan->dt = d.dtype, plan->batch = d.batch, plan->bias_dt = d.bias_dtype, plan->has_lengths = d.has_key_lengths != 0;
    plan->size = d.head_size <= 32 ? 32 : d.head_size <= 64 ? 64 : d.head_size <= 96 ? 96 : d.head_size <= 128 ? 128 : d.head_size <= 160 ? 160 : 256;
    plan->far = std::max(a.k_pt, a.v_pt) >= (1 << 24);
    const int64_t pairs = (int64_t)d.batch * d.kv_heads;
    const int cus = e.props.multiProcessorCount;
    const bool few = rows * pairs < 64ll * cus;
    plan->waves = few && plan->size <= ATT_ONE_WAVE ? 1 : 4;
    // Eight waves to a tile of keys where that leaves the fullest CU no more waves: half the trips into LDS (4096 x 4096 x 8 heads of
    // 64, batch 4: 146 and 157 us with eight and four; one CU's share the other way round, batch 5: 209 and 194).
    const auto fullest = [&](int waves) { return ((rows + 32 * waves - 1) / (32 * waves) * pairs + cus - 1) / cus * waves; };
    if (!few && plan->size % 64 == 0 && plan->size <= 128 && fullest(8) * 95 < fullest(4) * 100) plan->waves = 8;
    a.blocks = (int)((rows + 32 * plan->waves - 1) / (32 * plan->waves));
    a.splits = 1;
    const int tiles = (d.kv_len + ATT_KEYS - 1) / ATT_KEYS;
    // Two tiles at least to a part, parts for two workgroups to a CU.  The second kernel costs as much as four tiles one behind the
    // other.  (us, parts of 2, 4, 8 tiles: 1 query, 4096 keys, 8 key heads of 128: 12.6, 15.4, 22.3; all in one: 115.  5 tiles: 10.7 in
    // two parts, 9.4 in one.  2 x 2 key heads over 50176 keys: 28.9 with two workgroups to a CU, 32.5 and 36.2 with one and four)
    if (few && tiles >= 6) a.splits = (int)std::max<int64_t>(1, std::min<int64_t>((2 * cus + a.blocks * pairs - 1) / (a.blocks * pairs), std::min(tiles / 2, ATT_MOST_SPLITS)));
    check_grid(a.blocks * pairs * a.splits, 64 * plan->waves, "attention");
    a.total = (int)(a.blocks * pairs * a.splits);
    const int64_t scores = (int64_t)d.batch * d.q_heads * d.q_len * d.kv_len;
    const int64_t bias_size = d.bias_dtype == CLDNN_HIP_NO_TYPE ? 0 : d.bias_dtype == CLDNN_HIP_F32 ? 4 : 2;
    info.launches = a.splits > 1 ? 2 : 1, info.block = 64 * plan->waves, info.grid = a.total;
    info.lds_bytes = 4 * ATT_KEYS * plan->size * 2;
    if (a.splits > 1) info.workspace_bytes = pairs * a.splits * rows * (d.head_size + 2) * 4;
    info.ops = 4 * scores * d.head_size;
    info.bytes = 4ll * d.batch * d.head_size * ((int64_t)d.q_len * d.q_heads + (int64_t)d.kv_len * d.kv_heads)
                 + bias_size * (a.b_pb ? d.batch : 1) * (a.b_ph ? d.q_heads : 1) * (a.b_pq ? d.q_len : 1) * (int64_t)d.kv_len;
    snprintf(info.kernel_name, sizeof info.kernel_name, "attention<%d,%d wave%s%s%s>", plan->size, plan->waves, plan->waves > 1 ? "s" : "",
             plan->far ? ",far" : "", a.splits > 1 ? ",split keys" : "");
    return plan.release();
}

void attention_launch(hipStream_t s, const AttentionPlan& p, void* workspace, const void* q, const void* k, const void* v, const int32_t* lengths,
                      const void* bias, void* out)
{
    const AttentionArgs& a = p.a;
    const bool has_bias = p.bias_dt != CLDNN_HIP_NO_TYPE;
    CHIP_REQUIRE((!p.has_lengths || lengths) && (!has_bias || bias), CLDNN_HIP_INVALID_ARG, "null device pointer");
    check_aligned(q, 16, "q"), check_aligned(k, 16, "k"), check_aligned(v, 16, "v"), check_aligned(out, 16, "output");
    if (p.has_lengths) check_aligned(lengths, 4, "key_lengths");
    else lengths = nullptr;
    if (has_bias) check_aligned(bias, p.bias_dt == CLDNN_HIP_F32 ? 4 : 2, "bias");
    with_half(p.dt, [&](auto t) {
        typedef decltype(t) T;
        const auto launch = [&](auto d) {
            constexpr int D = decltype(d)::value;
            const auto with = [&](auto* of) {
                typedef typename std::remove_pointer<decltype(of)>::type B;
                const auto go = [&](auto f) {
                    hipLaunchKernelGGL(f, dim3(a.total), dim3(64 * p.waves), 0, s, a, (const T*)q, (const T*)k, (const T*)v, lengths, (const B*)bias, (T*)out, (float*)workspace);
                };
                if constexpr (D <= ATT_ONE_WAVE)
                    if (p.waves == 1) return go(p.far ? attention_kernel<T, D, B, 1, true> : attention_kernel<T, D, B, 1, false>);
                if constexpr (D % 64 == 0 && D <= 128)
                    if (p.waves == 8) return go(p.far ? attention_kernel<T, D, B, 8, true> : attention_kernel<T, D, B, 8, false>);
                go(p.far ? attention_kernel<T, D, B, 4, true> : attention_kernel<T, D, B, 4, false>);
            };
            if (!has_bias) with((void*)nullptr);
            else if (p.bias_dt == CLDNN_HIP_F32) with((float*)nullptr);
            else with((T*)nullptr);
        };
        switch (p.size) {
        case 32: launch(std::integral_constant<int, 32>()); break;
        case 64: launch(std::integral_constant<int, 64>()); break;
        case 96: launch(std::integral_constant<int, 96>()); break;
        case 128: launch(std::integral_constant<int, 128>()); break;
        case 160: launch(std::integral_constant<int, 160>()); break;
        default: launch(std::integral_constant<int, 256>());
        }
        if (a.splits > 1)
            hipLaunchKernelGGL((attention_join_kernel<T>), dim3(a.rows, p.a.total / a.blocks / a.splits), dim3(ATT_JOIN), 0, s, a, (const float*)workspace, (T*)out);
    });
    CHIP_CHECK(hipGetLastError());
}

void free_plan(AttentionPlan* p) { delete p; }

}  // namespace chip
