// vq2_select.hip -- expert routing with softmax or sigmoid scores, a balance
// bias, expert groups and weights that are renormalised or not (gfx950).
//
// Per token: s_e = softmax(l)_e or sigmoid(l_e), choice c_e = s_e + b_e; the
// groups (E / G consecutive experts) are ranked by their best c or the sum of
// their two best and the first `keep` stay; the k best c of the experts that
// stay are taken in descending order, ties to the lower id.  Weights come from
// s alone.  An expert whose logit is -inf or NaN (or whose choice is) is
// masked: it ranks behind every other one and weighs 0.
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
};

constexpr double KEY_MASKED = -1e300;

// Choice and expert in one double, so that one v_max_f64 compares both: the
// low 10 bits of the mantissa carry the id, such that the lower one wins among
// equal choices.  Choices are compared to 42 bits then; fp32 logits, compared
// themselves where scores order alike, have 24 and stay exact.
__device__ __forceinline__ double choice_key(double c, int e)
{
    // (+ 0.0: -0 is 0; no infinity, whose low bits make a NaN)
    uint64_t b = __builtin_bit_cast(uint64_t, fmin(c, 1e300) + 0.0) & ~1023ull;
    b |= (b >> 63) ? (uint64_t)e : (uint64_t)(1023 - e);
    return __builtin_bit_cast(double, b);
}

__device__ __forceinline__ int key_expert(double key)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, key);
    return (b >> 63) ? (int)(b & 1023) : 1023 - (int)(b & 1023);
}

__device__ __forceinline__ double wave_max_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmax(v, __shfl_xor(v, off));
    return v;
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// One wave per token; lane holds experts j * 64 + lane.
template <int LT, int RPL>
__global__ void __launch_bounds__(64) select_kernel(SelectArgs a)
{
    __shared__ double s_c[RPL * 64];
    const int lane = threadIdx.x;
    const int64_t t = blockIdx.x;
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
            s[j] = 1.0 / (1.0 + exp(-(double)l[j]));
        else
            s[j] = l[j] == m ? 1.0 : exp((double)l[j] - (double)m);
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
        __syncthreads();
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
    for (int j = 0; j < RPL; j++) {
        const int e = j * 64 + lane;
        key[j] = e < a.n_e && key[j] > -INFINITY ? choice_key(key[j], e) : -INFINITY;
    }
    int id = 0;
    for (int r = 0; r < a.k; r++) {
        double best = key[0];
#pragma unroll
        for (int j = 1; j < RPL; j++) best = fmax(best, key[j]);
        best = wave_max_f64(best);
#pragma unroll
        for (int j = 0; j < RPL; j++)
            if (key[j] == best) key[j] = -INFINITY;
        if (lane == r) id = key_expert(best);
    }
    // the weights: lane r takes choice r's logit again
    double sw = 0.0;
    if (lane < a.k) {
        float x = ld_t<LT>(a.logits, row + id);
        bool masked = !(x > -INFINITY);
        if (a.bias) masked |= !(a.bias[id] > -INFINITY);
        if (a.scoring == VQ2_SCORE_SIGMOID)
            sw = 1.0 / (1.0 + exp(-(double)x));
        else
            sw = (x == m ? 1.0 : exp((double)x - (double)m)) / z;
        if (masked) sw = 0.0;
    }
    const double tot = a.renorm ? wave_sum_f64(sw) : 1.0;
    const int slots = a.k + (a.shared_id >= 0 ? 1 : 0);
    if (lane < a.k) {
        a.ids[t * slots + lane] = id;
        a.w[t * slots + lane] = tot > 0.0 ? (float)(sw / tot * (double)a.scale) : 0.0f;
    }
    if (a.shared_id >= 0) {
        const float g = a.gate ? router_shared_weight(a.gate, a.g_dt, a.h, a.h_dt, t, a.hidden, lane) : 1.0f;
        if (lane == 0) {
            a.ids[t * slots + a.k] = (int32_t)a.shared_id;
            a.w[t * slots + a.k] = g;
        }
    }
}

template <int LT>
void launch_rpl(const SelectArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)a.tokens), block(64);
    if (a.n_e <= 64)
        hipLaunchKernelGGL((select_kernel<LT, 1>), grid, block, 0, st, a);
    else if (a.n_e <= 256)
        hipLaunchKernelGGL((select_kernel<LT, 4>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((select_kernel<LT, 16>), grid, block, 0, st, a);
}

}  // namespace

int router_select_launch(const RouterSelectCall& c)
{
    if (c.tokens == 0) return VQ2_OK;
    SelectArgs a{c.logits, c.l_stride, c.tokens,    (int)c.n_experts, c.k, c.scoring, c.n_groups, c.keep,
                 (int)(c.n_experts / c.n_groups),   c.group_score,    c.renorm, c.scale, c.bias, c.h, c.h_dt,
                 c.hidden, c.gate, c.g_dt, c.shared_id, c.ids, c.w};
    hipStream_t st = (hipStream_t)c.stream;
    if (c.l_dt == VQ2_DT_F32)
        launch_rpl<VQ2_DT_F32>(a, st);
    else if (c.l_dt == VQ2_DT_F16)
        launch_rpl<VQ2_DT_F16>(a, st);
    else
        launch_rpl<VQ2_DT_BF16>(a, st);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_hip_error(err, "vq2 router select launch");
    return VQ2_OK;
}

}  // namespace vq2
