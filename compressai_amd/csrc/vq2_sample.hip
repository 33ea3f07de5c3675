// vq2_sample.hip -- the next token from a row of logits and a given random
// number, under temperature, top-k, top-p and min-p (gfx950).
//
// Weights are w_i = exp((l_i - max) / temperature).  Entries are ordered by
// logit, descending, ties to the lower column; top-k keeps the first k of
// them, top-p those whose predecessors weigh less than p of what top-k kept,
// min-p those with w_i >= min_p.  The token is the first column at which the
// running sum of kept weights exceeds u times their total.
//
// Which token comes out hangs on sums over the whole row, so weights are
// computed in 64 bits and summed as integers of 2^-42: any order of
// summation gives the same total, and a result does not depend on how the
// row was split.  (A weight below 2^-43 of the largest counts as 0.)
#include "vq2_common.hpp"
#include "vq2_router.hpp"
#include "vq2_internal.hpp"

namespace vq2 {

namespace {

constexpr int NT = 1024;  // threads of a row's workgroup
constexpr double UNIT = 4398046511104.0;  // 2^42: one weight of 1

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab;
    const float* u;
    const float* temperature_rows;
    const int32_t* top_k_rows;
    const float* top_p_rows;
    const float* min_p_rows;
    float temperature, top_p, min_p;
    int64_t top_k;
    int64_t* out_idx;
    float* out_logprob;
};

// Order of a row's entries: larger is earlier.
__device__ __forceinline__ uint64_t order_key(float l, int i)
{
    return argmax_key(l + 0.0f, i);  // (+ 0: -0 is 0)
}

struct Weigher {
    float max;
    double inv_t;
    __device__ __forceinline__ double operator()(float l) const
    {
        if (l == max) return 1.0;
        const double w = exp(((double)l - (double)max) * inv_t);
        return l > -INFINITY && w > 0.0 ? w : 0.0;  // (NaN: 0)
    }
};

__device__ __forceinline__ uint64_t fixed(double w) { return (uint64_t)(w * UNIT + 0.5); }

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* s)
{
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
    for (int i = 0; i < NT / 64; i++) r += s[i];
    return r;
}

// The key of the last entry that stays when an entry stays while less than
// `limit` stands before it, among the entries whose key is at least `from`.
// amount(l) is what an entry counts.  0 if all stay.
template <int LT, class F>
__device__ uint64_t threshold(const SampleArgs& a, int64_t row, uint64_t from, uint64_t limit, F amount, uint64_t* hist,
                              uint64_t* s_pick)
{
    uint64_t prefix = 0, acc = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += NT) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < a.vocab; i += NT) {
            const float l = ld_t<LT>(a.logits, row + i);
            const uint64_t key = order_key(l, i);
            if (l > -INFINITY && key >= from && (shift == 56 || key >> (shift + 8) == prefix))
                atomicAdd((unsigned long long*)&hist[(key >> shift) & 255], (unsigned long long)amount(l));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255;
            for (; d >= 0 && acc + hist[d] < limit; d--) acc += hist[d];
            s_pick[0] = (uint64_t)(int64_t)d;
            s_pick[1] = acc;
        }
        __syncthreads();
        const int64_t d = (int64_t)s_pick[0];
        acc = s_pick[1];
        __syncthreads();
        if (d < 0) return 0;  // (only in the first round)
        prefix = prefix << 8 | (uint64_t)d;
    }
    return prefix;
}

template <int LT>
__global__ void __launch_bounds__(NT) sample_kernel(SampleArgs a)
{
    __shared__ uint64_t s_red[NT / 64], s_hist[256], s_pick[2];
    __shared__ float s_max[NT / 64];
    const int b = blockIdx.x, tid = threadIdx.x;
    const int64_t row = b * a.stride;
    const float temperature = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
    const int64_t top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
    const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
    const float min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;

    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += NT) m = fmaxf(m, ld_t<LT>(a.logits, row + i));
    m = wave_max_all(m);
    if ((tid & 63) == 0) s_max[tid >> 6] = m;
    __syncthreads();
    for (int i = 0; i < NT / 64; i++) m = fmaxf(m, s_max[i]);
    if (m == -INFINITY) {
        if (tid == 0) {
            a.out_idx[b] = -1;
            a.out_logprob[b] = NAN;
        }
        return;
    }
    const bool greedy = !(temperature > 0.0f);
    const Weigher weigh{m, greedy ? 1.0 : 1.0 / (double)temperature};
    uint64_t thr = 0;
    const uint64_t k = greedy ? 1 : top_k > 0 ? (uint64_t)top_k : 0;
    if (k > 0 && k < (uint64_t)a.vocab)
        thr = threshold<LT>(a, row, 0, k, [](float) { return 1ull; }, s_hist, s_pick);
    if (top_p < 1.0f) {
        uint64_t z = 0;
        for (int i = tid; i < a.vocab; i += NT) {
            const float l = ld_t<LT>(a.logits, row + i);
            if (order_key(l, i) >= thr) z += fixed(weigh(l));
        }
        z = block_sum(z, s_red);
        const uint64_t limit = top_p > 0.0f ? (uint64_t)fmax(1.0, ceil((double)top_p * (double)z)) : 1;
        const uint64_t t = threshold<LT>(a, row, thr, limit, [&](float l) { return fixed(weigh(l)); }, s_hist, s_pick);
        thr = t > thr ? t : thr;
    }
    auto kept = [&](int i) -> uint64_t {
        const float l = ld_t<LT>(a.logits, row + i);
        const double w = weigh(l);
        return l > -INFINITY && order_key(l, i) >= thr && w >= (double)fminf(min_p, 1.0f) ? fixed(w) : 0;
    };
    uint64_t total = 0;
    for (int i = tid; i < a.vocab; i += NT) total += kept(i);
    total = block_sum(total, s_red);
    const double at = fmin(fmax((double)a.u[b], 0.0), 1.0) * (double)total;
    uint64_t target = (uint64_t)at;
    if (target >= total) target = total - 1;
    // tiles of NT columns, each scanned
    uint64_t base = 0;
    for (int i0 = 0; i0 < a.vocab; i0 += NT) {
        const int i = i0 + tid;
        const uint64_t v = i < a.vocab ? kept(i) : 0;
        uint64_t run = v;
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t o = __shfl_up(run, off);
            if ((tid & 63) >= off) run += o;
        }
        __syncthreads();
        if ((tid & 63) == 63) s_red[tid >> 6] = run;
        __syncthreads();
        uint64_t all = 0;
        for (int w = 0; w < NT / 64; w++) {
            if (w == (tid >> 6)) run += all;
            all += s_red[w];
        }
        if (v > 0 && base + run > target && base + run - v <= target) {
            a.out_idx[b] = i;
            const double w = weigh(ld_t<LT>(a.logits, row + i));
            a.out_logprob[b] = (float)(log(w) - log((double)total / UNIT));
        }
        base += all;
        if (base > target) break;
    }
}

}  // namespace

size_t sample_workspace_bytes(int64_t, int64_t) { return 0; }

int sample_launch(const SampleCall& c)
{
    if (c.rows == 0) return VQ2_OK;
    SampleArgs a{c.logits, c.l_stride, (int)c.vocab, c.u, c.temperature_rows, c.top_k_rows, c.top_p_rows, c.min_p_rows,
                 c.temperature, c.top_p, c.min_p, c.top_k, c.out_idx, c.out_logprob};
    hipStream_t st = (hipStream_t)c.stream;
    const dim3 grid((unsigned)c.rows), block(NT);
    if (c.l_dt == VQ2_DT_F32)
        hipLaunchKernelGGL(sample_kernel<VQ2_DT_F32>, grid, block, 0, st, a);
    else if (c.l_dt == VQ2_DT_F16)
        hipLaunchKernelGGL(sample_kernel<VQ2_DT_F16>, grid, block, 0, st, a);
    else
        hipLaunchKernelGGL(sample_kernel<VQ2_DT_BF16>, grid, block, 0, st, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_hip_error(err, "vq2 sample launch");
    return VQ2_OK;
}

}  // namespace vq2
