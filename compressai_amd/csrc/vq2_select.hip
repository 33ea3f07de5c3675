// vq2_select.hip -- expert routing with softmax or sigmoid scores, a balance
// bias, expert groups and weights that are renormalised or not (gfx950).
//
// Per token: s_e = softmax(l)_e or sigmoid(l_e), choice c_e = s_e + b_e; the
// groups (E / G consecutive experts) are ranked by their best c or the sum of
// their two best and the first `keep` stay; the k best c of the experts that
// stay are taken in descending order, ties to the lower id.  Weights come from
// s alone.  An expert whose logit is -inf or NaN (or whose choice is) is
// masked: it ranks behind every other one and weighs 0.  Without a bias c
// orders as the logits do, which are compared themselves.
//
// Choices that differ in the eighth digit must not trade places, so they are
// made in 64 bits; but a sigmoid of 64 bits for each of E experts costs several
// times what the rest does.  Two kernels:
//   rows   16 lanes a token, four tokens a wave.  Choices of 32 bits, cut to
//          23 to 26 bits of their range with the expert's id below them, make
//          one word each: a lane sorts its own (a network of v_min / v_max_u32),
//          rounds of a maximum over the 16 lanes (DPP) take the k + 2 best, and
//          only those are computed in 64 bits and put in order by them.  The
//          words of what was left out say whether any of it could belong among
//          the k (or whether two groups are too close to tell): such tokens, and
//          those with too few experts, go to
//   token  one wave a token, all of it in 64 bits.
//
// Kernel times on MI355X, us, of the rows kernel | the token kernel:
//   1 token, 256 experts fp32, sigmoid, bias, 4 of 8 groups, gate    7.7 |   7.4
//   64 tokens, 64 experts bf16, softmax                              3.9 |   4.3
//   333 tokens, 160 experts fp32, softmax, 3 of 8 groups             8.0 |   7.2
//   4096 tokens, 256 experts fp16, sigmoid, gate over 2048 (19 MB)  10.0 |    11
//   16384 tokens, 256 experts bf16, sigmoid, bias, 4 of 8 groups    15.0 |    36
//   32768 tokens, 512 experts fp32, sigmoid, bias (67 MB)           30.3 |   164
// The rows kernel takes every call it has room for (512 experts, 12 of them
// chosen, 16 groups: candidates, groups and a lane's words in 16 lanes).  Up to
// some 500 tokens the token kernel is the faster one where there is a bias or a
// gate (16 tokens of 256 experts bf16: 6.0 | 5.5, 7.7 | 5.8) and the slower one
// without (4.8 | 5.4) or with 512 experts (7.3 | 11); but the two round weights
// differently, and a limit between them would make a token's last bits depend on
// how many others are routed with it.
// Few tokens are bound by the chain of a wave (loads, sort, k + 2 rounds, 64-bit
// candidates: 4 to 8 us); many by its vector instructions, which issue in 84 % of
// the cycles of the last line and in 74 % of the one above: 51 an expert in the
// last line, of which the sorting network of 32 words a lane is 10, and 2.2 TB/s
// of the 4.9 that a large copy reaches.
// Choices of 32 bits tell little apart where one expert's lies far from all
// others: unbiased fp32 logits masked by a large finite number (-1e9, the type's
// lowest) share one place, and every token goes on to 64 bits, four in turn in a
// wave.  4096 tokens of 256 experts, half of them masked so: 24 us, against 5.7
// with -inf or without masks and 9.8 by the token kernel alone.  (So does a bias
// far below all others; 16-bit logits without a bias order exactly.)
#include "vq2_common.hpp"
#include "vq2_router.hpp"
#include "vq2_internal.hpp"

namespace vq2 {

namespace {

struct SelectArgs {
    const void* logits;
    int64_t stride, tokens;
    int n_e, k, scoring, n_groups, keep, group_size, group_score, renorm;
    float scale;
    const float* bias;
    const void* h;
    int h_dt;
    int64_t hidden;
    const void* gate;
    int g_dt;
    int64_t shared_id;
    int32_t* ids;
    float* w;
    __device__ __forceinline__ int slots() const { return k + (shared_id >= 0 ? 1 : 0); }
};

// Scores of 64 bits: exp for x <= 0, down to the steps of 2^-1074 that 64 bits
// end in, and the sigmoid, 0 where e^-x is none of 64 bits.
__device__ __forceinline__ double exp_f64(double x)
{
    uint32_t whole;
    const double p = exp2_f64_fraction(fmax(x * LOG2E_F64, -1100.0), whole);
    return __builtin_amdgcn_ldexp(p, (int)whole);
}
// 1 / x of a normal x whose reciprocal is normal, to 2^-51: the instruction's
// approximation and two Newton steps
__device__ __forceinline__ double reciprocal_f64(double x)
{
    double r = __builtin_amdgcn_rcp(x);
    r = fma(fma(-x, r, 1.0), r, r);
    return fma(fma(-x, r, 1.0), r, r);
}
__device__ __forceinline__ double sigmoid_f64(double x)
{
    const double e = exp_f64(-fabs(x)), r = reciprocal_f64(1.0 + e);
    return x >= 0.0 ? r : x >= -709.78271289338397 ? e * r : 0.0;
}

// LDS written by a wave's lanes is read by its others.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ------------------------------------------------- sigmoid(gate . h) of a token
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8])
{
    typedef u32x4 __attribute__((aligned(2))) any_t;
    if constexpr (DT == VQ2_DT_F32) {
        const u32x4 a = *(const any_t*)((const float*)p + i), b = *(const any_t*)((const float*)p + i + 4);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = __uint_as_float(a[j]);
            v[4 + j] = __uint_as_float(b[j]);
        }
    } else {
        const u32x4 a = *(const any_t*)((const uint16_t*)p + i);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t h = j & 1 ? a[j / 2] >> 16 : a[j / 2] & 0xFFFFu;
            v[j] = DT == VQ2_DT_F16 ? f16_bits_to_f32((uint16_t)h) : bf16_bits_to_f32(h);
        }
    }
}

template <int GT, int HT>
__device__ __forceinline__ float gate_dot(const SelectArgs& a, int64_t t, int lane)
{
    const int64_t row = t * a.hidden, whole = a.hidden / 512 * 512;
    float d = 0.0f;
#pragma unroll 4
    for (int64_t i = lane * 8; i < whole; i += 512) {
        float g[8], x[8];
        load8<GT>(a.gate, i, g);
        load8<HT>(a.h, row + i, x);
#pragma unroll
        for (int j = 0; j < 8; j++) d = fmaf(g[j], x[j], d);
    }
    for (int64_t i = whole + lane; i < a.hidden; i += 64) d = fmaf(ld_t<GT>(a.gate, i), ld_t<HT>(a.h, row + i), d);
    return wave_sum_all(d);
}

// the shared expert's weight, uniform over the wave
__device__ __forceinline__ float shared_weight(const SelectArgs& a, int64_t t, int lane)
{
    if (!a.gate) return 1.0f;
    float d;
    switch (a.g_dt * 3 + a.h_dt) {
    case VQ2_DT_F32 * 3 + VQ2_DT_F32: d = gate_dot<VQ2_DT_F32, VQ2_DT_F32>(a, t, lane); break;
    case VQ2_DT_F32 * 3 + VQ2_DT_F16: d = gate_dot<VQ2_DT_F32, VQ2_DT_F16>(a, t, lane); break;
    case VQ2_DT_F32 * 3 + VQ2_DT_BF16: d = gate_dot<VQ2_DT_F32, VQ2_DT_BF16>(a, t, lane); break;
    case VQ2_DT_F16 * 3 + VQ2_DT_F32: d = gate_dot<VQ2_DT_F16, VQ2_DT_F32>(a, t, lane); break;
    case VQ2_DT_F16 * 3 + VQ2_DT_F16: d = gate_dot<VQ2_DT_F16, VQ2_DT_F16>(a, t, lane); break;
    case VQ2_DT_F16 * 3 + VQ2_DT_BF16: d = gate_dot<VQ2_DT_F16, VQ2_DT_BF16>(a, t, lane); break;
    case VQ2_DT_BF16 * 3 + VQ2_DT_F32: d = gate_dot<VQ2_DT_BF16, VQ2_DT_F32>(a, t, lane); break;
    case VQ2_DT_BF16 * 3 + VQ2_DT_F16: d = gate_dot<VQ2_DT_BF16, VQ2_DT_F16>(a, t, lane); break;
    default: d = gate_dot<VQ2_DT_BF16, VQ2_DT_BF16>(a, t, lane); break;
    }
    return 1.0f / (1.0f + __expf(-d));
}

// ------------------------------------------------------------- one wave a token
constexpr double KEY_MASKED = -1e300;

template <int CTRL>
__device__ __forceinline__ double row_f64(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp_mov<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_mov<CTRL>((int)(uint32_t)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// (a round's chain is mostly this: within a row of 16 by rotations, then two
// shuffles)
__device__ __forceinline__ double wave_max_f64(double v)
{
    v = fmax(v, row_f64<0x128>(v));
    v = fmax(v, row_f64<0x124>(v));
    v = fmax(v, row_f64<0x122>(v));
    v = fmax(v, row_f64<0x121>(v));
    v = fmax(v, __shfl_xor(v, 16));
    return fmax(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// A token's choice by a whole wave; lane holds experts j * 64 + lane, s_c is
// RPL * 64 doubles of LDS of the wave's own.
template <int LT, int RPL>
__device__ void select_token(const SelectArgs& a, int64_t t, int lane, double* s_c)
{
    const int64_t row = t * a.stride;
    float l[RPL];
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        const int e = j * 64 + lane;
        l[j] = ld_t<LT>(a.logits, row + (e < a.n_e ? e : 0));
        if (e >= a.n_e || !(l[j] > -INFINITY)) l[j] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < RPL; j++) m = fmaxf(m, l[j]);
    m = wave_max_all(m);
    double z = 0.0, s[RPL];
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        if (a.scoring == VQ2_SCORE_SIGMOID)
            s[j] = sigmoid_f64((double)l[j]);
        else
            s[j] = l[j] == m ? 1.0 : exp_f64((double)l[j] - (double)m);
        if (l[j] == -INFINITY) s[j] = 0.0;
        z += s[j];
    }
    if (a.scoring == VQ2_SCORE_SOFTMAX) {
        z = wave_sum_f64(z);
#pragma unroll
        for (int j = 0; j < RPL; j++) s[j] /= z;
    }
    // without a bias choices order as the logits, which do not round together
    double key[RPL];
#pragma unroll
    for (int j = 0; j < RPL; j++) {
        const int e = j * 64 + lane;
        double c = s[j] + (a.bias && e < a.n_e ? (double)a.bias[e] : 0.0);
        if (l[j] == -INFINITY || !(c > -INFINITY)) c = KEY_MASKED;
        key[j] = a.bias || c == KEY_MASKED ? c : (double)l[j];
        s[j] = a.group_score == VQ2_GROUP_TOP2 ? c : key[j];
    }
    if (a.n_groups > 1) {
#pragma unroll
        for (int j = 0; j < RPL; j++) s_c[j * 64 + lane] = s[j];
        wave_sync();
        double g1 = -INFINITY, g2 = -INFINITY;
        if (lane < a.n_groups) {
            for (int i = 0; i < a.group_size; i++) {
                const double c = s_c[lane * a.group_size + i];
                g2 = fmax(g2, fmin(g1, c));
                g1 = fmax(g1, c);
            }
            if (a.group_score == VQ2_GROUP_TOP2 && g2 > KEY_MASKED) g1 += g2;
        }
        int rank = 0;
        for (int g = 0; g < a.n_groups; g++) {
            const double o = __shfl(g1, g);
            rank += o > g1 || (o == g1 && g < lane);
        }
        const uint64_t stay = __ballot(lane < a.n_groups && rank < a.keep);
#pragma unroll
        for (int j = 0; j < RPL; j++) {
            const int e = j * 64 + lane;
            if (e < a.n_e && !((stay >> (e / a.group_size)) & 1)) key[j] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < RPL; j++)
        if (j * 64 + lane >= a.n_e) key[j] = -INFINITY;
    // the largest choice, and of its experts the lowest (choices that differ in
    // their last bit alone are told apart: sigmoids close to 1 do); `mine` is
    // the lane's first expert with it
    int id = 0;
    for (int r = 0; r < a.k; r++) {
        double best = key[0];
#pragma unroll
        for (int j = 1; j < RPL; j++) best = fmax(best, key[j]);
        best = wave_max_f64(best);
        int mine = RPL;
#pragma unroll
        for (int j = RPL - 1; j >= 0; j--)
            if (key[j] == best) mine = j;
        const uint64_t equal = __ballot(mine < RPL);
        const int first = __builtin_ctzll(equal);
        int at = __builtin_amdgcn_readlane(mine, first) * 64 + first;
        if (equal & (equal - 1)) {
#pragma unroll
            for (int j = RPL - 1; j >= 0; j--) {
                const uint64_t here = __ballot(mine == j);
                if (here) at = j * 64 + __builtin_ctzll(here);
            }
        }
#pragma unroll
        for (int j = 0; j < RPL; j++)
            if (j * 64 + lane == at) key[j] = -INFINITY;
        if (lane == r) id = at;
    }
    // the weights: lane r takes choice r's logit again
    double sw = 0.0;
    if (lane < a.k) {
        const float x = ld_t<LT>(a.logits, row + id);
        bool masked = !(x > -INFINITY);
        if (a.bias) masked |= !(a.bias[id] > -INFINITY);
        if (a.scoring == VQ2_SCORE_SIGMOID)
            sw = sigmoid_f64((double)x);
        else
            sw = (x == m ? 1.0 : exp_f64((double)x - (double)m)) / z;
        if (masked) sw = 0.0;
    }
    const double tot = a.renorm ? wave_sum_f64(sw) : 1.0;
    if (lane < a.k) {
        a.ids[t * a.slots() + lane] = id;
        a.w[t * a.slots() + lane] = tot > 0.0 ? (float)(sw / tot * (double)a.scale) : 0.0f;
    }
}

__device__ __forceinline__ void write_shared(const SelectArgs& a, int64_t t, int lane)
{
    const float g = shared_weight(a, t, lane);
    if (lane == 0) {
        a.ids[t * a.slots() + a.k] = (int32_t)a.shared_id;
        a.w[t * a.slots() + a.k] = g;
    }
}

template <int LT, int RPL>
__global__ void __launch_bounds__(64) select_token_kernel(SelectArgs a)
{
    __shared__ double s_c[RPL * 64];
    select_token<LT, RPL>(a, blockIdx.x, threadIdx.x, s_c);
    if (a.shared_id >= 0) write_shared(a, blockIdx.x, threadIdx.x);
}

// ----------------------------------------------------------- 16 lanes a token
constexpr int ROWS_MAX_E = 512, ROWS_MAX_K = 12, ROWS_MAX_G = 16;
constexpr int EXTRA = 2;  // candidates beyond k

template <int CTRL>
__device__ __forceinline__ float row_f32(float v)
{
    return __int_as_float(dpp_mov<CTRL>(__float_as_int(v)));
}
// Over the 16 lanes of a row (rotations by 8, 4, 2, 1), in all of them.
__device__ __forceinline__ float row_max(float v)
{
    v = fmaxf(v, row_f32<0x128>(v));
    v = fmaxf(v, row_f32<0x124>(v));
    v = fmaxf(v, row_f32<0x122>(v));
    return fmaxf(v, row_f32<0x121>(v));
}
__device__ __forceinline__ float row_min(float v) { return -row_max(-v); }
__device__ __forceinline__ float row_sum(float v)
{
    v += row_f32<0x128>(v);
    v += row_f32<0x124>(v);
    v += row_f32<0x122>(v);
    return v + row_f32<0x121>(v);
}
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v)
{
    v = max(v, (uint32_t)dpp_mov<0x128>((int)v));
    v = max(v, (uint32_t)dpp_mov<0x124>((int)v));
    v = max(v, (uint32_t)dpp_mov<0x122>((int)v));
    return max(v, (uint32_t)dpp_mov<0x121>((int)v));
}
__device__ __forceinline__ double row_sum(double v)
{
    v += row_f64<0x128>(v);
    v += row_f64<0x124>(v);
    v += row_f64<0x122>(v);
    return v + row_f64<0x121>(v);
}

// Descending, by odd-even merges.
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&v)[N])
{
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t x = v[i + j], y = v[i + j + k];
                        v[i + j] = max(x, y);
                        v[i + j + k] = min(x, y);
                    }
}

// Four tokens a wave, N experts a lane; four waves a workgroup.
template <int LT, int N, bool GROUPS, bool GATE>
__global__ void __launch_bounds__(256, 4) select_rows_kernel(SelectArgs a)
{
    constexpr int V = LT == VQ2_DT_F32 ? 4 : (N < 8 ? N : 8);  // experts of one load
    constexpr int IDB = N <= 4 ? 6 : N <= 8 ? 7 : N <= 16 ? 8 : 9, QB = 32 - IDB;
    constexpr uint32_t IDS = (1u << IDB) - 1;
    constexpr int HEADS = N < ROWS_MAX_K + EXTRA ? N : ROWS_MAX_K + EXTRA;
    constexpr int PER_TOKEN = 16 * N + ROWS_MAX_G;  // a group's scores are one apart from the next one's
    __shared__ uint32_t s_heads[4][HEADS * 64];
    __shared__ union {
        float c[4][GROUPS ? PER_TOKEN : 1];
        double token[GROUPS ? 16 * N : 1];  // (only groups take a whole wave there)
    } s_g[4];  // one a wave
    __shared__ float s_score[4][4][GROUPS ? 16 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane & 15, quarter = lane >> 4;
    const uint32_t tokens = (uint32_t)a.tokens, t0 = (blockIdx.x * 4 + wave) * 4;
    if (t0 >= tokens) return;
    const uint32_t t = t0 + quarter;
    const int64_t row = min(t, tokens - 1) * a.stride;
    const bool softmax = a.scoring == VQ2_SCORE_SOFTMAX, biased = a.bias != nullptr;
    const bool by_score = biased || (GROUPS && a.group_score == VQ2_GROUP_TOP2);
    // unbiased logits of 16 bits and an id fit a word: no candidate is in doubt
    const bool exact = LT != VQ2_DT_F32 && !biased;

    auto expert = [&](int j) { return ((j / V) * 16 + sub) * V + j % V; };
    const uint32_t magic = ((1u << 20) + a.group_size - 1) / a.group_size;
    auto group = [&](int e) { return (int)((uint32_t)e * magic >> 20); };  // (e / group_size, for e < 512)
    float l[N];
#pragma unroll
    for (int c = 0; c < N / V; c++) {
        const int e0 = expert(c * V);
        if (e0 + V <= a.n_e) {
            if constexpr (LT == VQ2_DT_F32) {
                typedef u32x4 __attribute__((aligned(4))) any_t;
                const u32x4 w = *(const any_t*)((const float*)a.logits + row + e0);
#pragma unroll
                for (int j = 0; j < 4; j++) l[c * V + j] = __uint_as_float(w[j]);
            } else {
                typedef uint32_t words_t __attribute__((ext_vector_type(V / 2)));
                typedef words_t __attribute__((aligned(2))) any_t;
                const words_t w = *(const any_t*)((const uint16_t*)a.logits + row + e0);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const uint32_t h = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
                    l[c * V + j] = LT == VQ2_DT_F16 ? f16_bits_to_f32((uint16_t)h) : bf16_bits_to_f32(h);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                l[c * V + j] = e0 + j < a.n_e ? ld_t<LT>(a.logits, row + e0 + j) : -INFINITY;
        }
    }
    // adds the biases of V experts
    auto add_bias = [&](int o, float* c) {
        const int e0 = expert(o * V);
#pragma unroll
        for (int j = 0; j < V; j += 4)
            if (e0 + j + 4 <= a.n_e) {
                typedef float f32x4 __attribute__((ext_vector_type(4)));
                typedef f32x4 __attribute__((aligned(4))) any_t;
                const f32x4 b = *(const any_t*)(a.bias + e0 + j);
#pragma unroll
                for (int i = 0; i < 4; i++) c[j + i] += b[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) c[j + i] += e0 + j + i < a.n_e ? a.bias[e0 + j + i] : 0.0f;
            }
    };
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (!(l[j] > -INFINITY)) l[j] = -INFINITY;  // (NaN)
        m = fmaxf(m, l[j]);
    }
    m = row_max(m);
    double z = 1.0;
    if (softmax && (biased || !a.renorm)) {
        z = 0.0;
#pragma unroll
        for (int j = 0; j < N; j++) z += exp_f64((double)l[j] - (double)m);  // (-inf and NaN: 0)
        z = row_sum(z);
    }

    // c: choices of 32 bits, -inf where masked
    float c[N];
    if (by_score) {
        if (softmax) {
            float z = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++) {
                c[j] = __builtin_amdgcn_exp2f((l[j] - m) * 1.44269504f);
                z += c[j];
            }
            const float r = 1.0f / row_sum(z);
#pragma unroll
            for (int j = 0; j < N; j++) c[j] *= r;
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) c[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -1.44269504f));
        }
        if (biased) {
#pragma unroll
            for (int o = 0; o < N / V; o++) add_bias(o, c + o * V);
        }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (l[j] == -INFINITY || !(c[j] > -INFINITY)) c[j] = -INFINITY;
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) c[j] = l[j];
    }
    // What a choice of 32 bits is off by, in units of its size or 1.  Sigmoid:
    // s (1 - s) |l| 1.5 steps of 2^-24 by the exponential's argument, s (1 - s) 2 by
    // the exponential, 3 by the sum and the reciprocal, 1 by the bias's addition:
    // 5 together.  Softmax: 1 by the argument, 38 by the sum of up to 32 + 4
    // terms, 4 by the rest.
    const float EPS = softmax ? 2.6e-6f : 3.5e-7f;
    bool unsure = softmax && !(m < INFINITY);
    uint32_t stays = 0xFFFFu;
    if constexpr (GROUPS) {
        float size = 1.0f;
#pragma unroll
        for (int j = 0; j < N; j++) size = fmaxf(size, c[j] == -INFINITY ? 0.0f : fabsf(c[j]));
        const float eps = EPS * row_max(size);
        float* const sc = s_g[wave].c[quarter];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int e = expert(j);
            if (e < a.n_e) sc[e + group(e)] = c[j];
        }
        wave_sync();
        // the lanes of a row share the groups: 1, 2, 4, 8 or 16 a group
        const int shift = a.n_groups > 8 ? 0 : a.n_groups > 4 ? 1 : a.n_groups > 2 ? 2 : 3, g = sub >> shift;
        float g1 = -INFINITY, g2 = -INFINITY;
        if (g < a.n_groups)
#pragma unroll 4
            for (int i = sub & ((1 << shift) - 1); i < a.group_size; i += 1 << shift) {
                const float x = sc[g * (a.group_size + 1) + i];
                g2 = fmaxf(g2, fminf(g1, x));
                g1 = fmaxf(g1, x);
            }
        auto merge = [&](float o1, float o2) {
            g2 = fmaxf(fminf(g1, o1), fmaxf(g2, o2));
            g1 = fmaxf(g1, o1);
        };
        if (shift >= 1) merge(dpp_xor1(g1), dpp_xor1(g2));
        if (shift >= 2) merge(dpp_xor2(g1), dpp_xor2(g2));
        if (shift >= 3) merge(dpp_half_mirror(g1), dpp_half_mirror(g2));
        if (a.group_score == VQ2_GROUP_TOP2 && g2 > -INFINITY) g1 += g2;
        float* const scores = s_score[wave][quarter];
        if ((sub & ((1 << shift) - 1)) == 0) scores[g] = g1;
        wave_sync();
        int rank = 0;
#pragma unroll 4
        for (int o = 0; o < a.n_groups; o++) {
            const float x = scores[o];
            rank += x > g1 || (x == g1 && o < g);
        }
        const bool real = g < a.n_groups, in = real && rank < a.keep;
        // groups closer than their scores are exact (logits are)
        const float lowest_in = row_min(in ? g1 : INFINITY), highest_out = row_max(real && !in ? g1 : -INFINITY);
        unsure |= by_score && highest_out > -INFINITY && !(lowest_in - highest_out > 4.0f * eps);
        const uint32_t lanes = (uint32_t)(__ballot(in) >> (quarter * 16)) & 0xFFFFu;
        stays = 0;
        for (int o = 0; o < a.n_groups; o++) stays |= (lanes >> (o << shift) & 1) << o;
        if (!biased) {  // the experts' own order is the logits'
#pragma unroll
            for (int j = 0; j < N; j++) c[j] = l[j];
        }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (!(stays >> group(expert(j)) & 1)) c[j] = -INFINITY;
    }
    float cmax = -INFINITY, cmin = INFINITY;
#pragma unroll
    for (int j = 0; j < N; j++) {
        cmax = fmaxf(cmax, c[j]);
        cmin = fminf(cmin, c[j] == -INFINITY ? INFINITY : c[j]);
    }
    cmax = row_max(cmax);
    cmin = row_min(cmin);
    const float range = cmax - cmin, scale = 0.9999f * (float)(1u << QB) / range;
    unsure |= !exact && !(range > 0.0f && range < INFINITY && scale < INFINITY);

    // words: place in the range, then the id, lower ids above
    uint32_t key[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        uint32_t place;
        if (exact) {  // the logit's own 16 bits, in their order (fp16's are fp32's top 19, zeros below)
            uint32_t u;
            if constexpr (LT == VQ2_DT_F16) u = __builtin_bit_cast(uint16_t, (_Float16)(c[j] + 0.0f));
            else u = __float_as_uint(c[j] + 0.0f) >> 16;
            place = u & 0x8000u ? 0xFFFFu - u : 0x8000u + u;
        } else {
            place = (uint32_t)((c[j] - cmin) * scale) + 1u;
        }
        key[j] = c[j] == -INFINITY ? 0u : place << IDB | (IDS - (uint32_t)expert(j));
    }
    sort_down(key);
#pragma unroll
    for (int j = 0; j < HEADS; j++) s_heads[wave][j * 64 + lane] = key[j];
    const int C = a.k + (exact ? 0 : EXTRA);
    uint32_t mine = 0, head = key[0], second = key[1], last = 0;
    int next = 2;
    for (int r = 0; r < C; r++) {
        last = row_max_u32(head);
        if (sub == r) mine = last;
        if (head == last) {
            head = second;
            second = next < HEADS ? s_heads[wave][next * 64 + lane] : 0;
            next++;
        }
    }

    // the candidates in 64 bits, one a lane
    const bool has = mine != 0;
    const int id = has ? (int)(IDS - (mine & IDS)) : 0;
    const float x = ld_t<LT>(a.logits, row + id);
    const double s = softmax ? exp_f64((double)x - (double)m) * (z == 1.0 ? 1.0 : reciprocal_f64(z)) : sigmoid_f64((double)x);
    const double choice = biased ? s + (double)a.bias[id] : (double)x;
    // they are nearly always in order already: then a candidate's rank is its lane
    int rank = sub;
    const int hid = has ? id : -1;
    auto ahead = [&](double o, int oid) { return oid >= 0 && (o > choice || (o == choice && oid < id)); };
    if (__ballot(has && ahead(row_f64<0x101>(choice), sub == 15 ? -1 : dpp_mov<0x101>(hid)))) {
        rank = 0;
#define VQ2_ROTATE(n) rank += ahead(row_f64<0x120 + n>(choice), dpp_mov<0x120 + n>(hid));
        VQ2_ROTATE(1) VQ2_ROTATE(2) VQ2_ROTATE(3) VQ2_ROTATE(4) VQ2_ROTATE(5) VQ2_ROTATE(6) VQ2_ROTATE(7) VQ2_ROTATE(8)
        VQ2_ROTATE(9) VQ2_ROTATE(10) VQ2_ROTATE(11) VQ2_ROTATE(12) VQ2_ROTATE(13) VQ2_ROTATE(14) VQ2_ROTATE(15)
#undef VQ2_ROTATE
    }
    const bool wins = has && rank < a.k;
    const float winners = row_sum(wins ? 1.0f : 0.0f);
    unsure |= winners < (float)a.k;
    if (!exact) {
        // `last` is the lowest candidate's word: what was left out is not above it.
        // Places are off by the choices' error and by the rounding of the
        // difference and the product (2^-23 of the range together, two of them).
        const float slack = 4.0f + (float)(QB > 23 ? 4u << (QB - 23) : 4u);
        const float margin = slack + (biased ? 2.0f * EPS * fmaxf(1.0f, fmaxf(fabsf(cmax), fabsf(cmin))) * scale : 0.0f);
        const float lowest = row_min(wins ? (float)(mine >> IDB) : INFINITY);
        unsure |= last != 0 && !(lowest - (float)(last >> IDB) > margin);
    }

    const double tot = a.renorm ? row_sum(wins ? s : 0.0) : 1.0;
    unsure |= !(tot > 1e-290);  // (no normal reciprocal)
    if (wins && !unsure && t < tokens) {
        a.ids[(int64_t)t * a.slots() + rank] = id;
        a.w[(int64_t)t * a.slots() + rank] = (float)(s * reciprocal_f64(tot) * (double)a.scale);
    }
    // the tokens that are left, by the whole wave
    const uint64_t left = __ballot(unsure && t < tokens);
    for (int q = 0; q < 4; q++)
        if (left >> (16 * q) & 1) {
            wave_sync();
            select_token<LT, (N + 3) / 4>(a, t0 + q, lane, s_g[wave].token);
        }
    if constexpr (GATE) {
        for (int q = 0; q < 4 && t0 + q < tokens; q++) write_shared(a, t0 + q, lane);
    } else if (a.shared_id >= 0 && sub == 0 && t < tokens) {
        a.ids[(int64_t)t * a.slots() + a.k] = (int32_t)a.shared_id;
        a.w[(int64_t)t * a.slots() + a.k] = 1.0f;
    }
}

template <int LT, int N, bool GROUPS>
void launch_rows(const SelectArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)((a.tokens + 15) / 16)), block(256);
    if (a.shared_id >= 0 && a.gate)
        hipLaunchKernelGGL((select_rows_kernel<LT, N, GROUPS, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((select_rows_kernel<LT, N, GROUPS, false>), grid, block, 0, st, a);
}

template <int LT, int N>
void launch_rows(const SelectArgs& a, hipStream_t st)
{
    return a.n_groups > 1 ? launch_rows<LT, N, true>(a, st) : launch_rows<LT, N, false>(a, st);
}

template <int LT>
void launch(const SelectArgs& a, hipStream_t st)
{
    if (a.n_e <= ROWS_MAX_E && a.k <= ROWS_MAX_K && a.n_groups <= ROWS_MAX_G) {
        if (a.n_e <= 64) return launch_rows<LT, 4>(a, st);
        if (a.n_e <= 128) return launch_rows<LT, 8>(a, st);
        if (a.n_e <= 256) return launch_rows<LT, 16>(a, st);
        return launch_rows<LT, 32>(a, st);
    }
    const dim3 grid((unsigned)a.tokens), block(64);
    if (a.n_e <= 64)
        hipLaunchKernelGGL((select_token_kernel<LT, 1>), grid, block, 0, st, a);
    else if (a.n_e <= 256)
        hipLaunchKernelGGL((select_token_kernel<LT, 4>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((select_token_kernel<LT, 16>), grid, block, 0, st, a);
}

}  // namespace

int router_select_launch(const RouterSelectCall& c)
{
    if (c.tokens == 0) return VQ2_OK;
    SelectArgs a{c.logits, c.l_stride, c.tokens,    (int)c.n_experts, c.k, c.scoring, c.n_groups, c.keep,
                 (int)(c.n_experts / c.n_groups),   c.group_score,    c.renorm, c.scale, c.bias, c.h, c.h_dt,
                 c.hidden, c.gate, c.g_dt, c.shared_id, c.ids, c.w};
    // all groups staying is no grouping
    if (a.keep == a.n_groups) a.n_groups = a.keep = 1, a.group_size = a.n_e;
    hipStream_t st = (hipStream_t)c.stream;
    if (c.l_dt == VQ2_DT_F32)
        launch<VQ2_DT_F32>(a, st);
    else if (c.l_dt == VQ2_DT_F16)
        launch<VQ2_DT_F16>(a, st);
    else
        launch<VQ2_DT_BF16>(a, st);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_hip_error(err, "vq2 router select launch");
    return VQ2_OK;
}

}  // namespace vq2
