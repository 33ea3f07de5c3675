// vq2_sample.hip -- the next token from a row of logits and a given random
// number, under temperature, top-k, top-p and min-p (gfx950).
//
// Weights are w_i = exp((l_i - max) / temperature).  Entries are ordered by
// logit, descending, ties to the lower column; top-k keeps the first k of
// them, top-p those whose predecessors weigh less than p of what top-k kept,
// min-p those with w_i >= min_p.  The token is the first column at which the
// running sum of kept weights exceeds u times their total.
//
// Which token comes out hangs on sums over a whole row, and two draws differ
// by as little as one flat row's weight, 1e-5 of the total: in 32 bits one
// draw in some hundred would be another.  So weights are computed in 64 bits
// (exp2_f64), and where entries are put in order they are summed as whole
// numbers of 2^-42 of the largest (a weight below 2^-43 counts as 0), whose
// sum is the same in any order.
//
// Three launches:
//   stats    A row is cut into units, each a contiguous piece that one wave
//            reads; every unit's maximum and weight (for top-k, the maxima of
//            finer groups).
//   collect  The row's maximum and total are known from the units and with
//            them a logit below which nothing can stay:
//              top-k  the k-th largest of the groups' maxima (k entries are
//                     that large);
//              top-p  w < (1 - p) Z / V: all such entries together weigh less
//                     than (1 - p) Z, which the last entries may be short of;
//              min-p  w < min_p;  always: w < 2^-45.
//            The entries above, usually some hundred to some thousand of a
//            row, are listed in column order.
//   finish   One workgroup a row, on the list in LDS: up to 256 entries are
//            ranked directly, more are narrowed down by histograms; a running
//            sum over the list finds the token.
// A draw without a border (no top-k, top-p or min-p) needs no list: the unit
// whose weights' running sum passes u Z is read again (two launches).  A row
// with too many entries for LDS (flat rows) has a histogram of each slice of
// 8 units beside the lists: the finish adds them up, fetches the entries of
// the border's bin alone and, at the end, the slice that the draw falls into.
// Long ties in that bin are the one case that is finished entry by entry.
#include <float.h>

#include "vq2_common.hpp"
#include "vq2_router.hpp"
#include "vq2_internal.hpp"

namespace vq2 {

namespace {

constexpr int NT = 512;           // threads of a workgroup
constexpr int NW = NT / 64;       // its waves, one unit each: a slice
constexpr int MAX_UNITS = 1024;   // units of a row
constexpr int MAX_SLICES = MAX_UNITS / NW;
constexpr int LIST = 3072;        // entries of the list in LDS
constexpr int DIRECT = 256;       // entries that are ranked directly
constexpr int BINS = 256;         // of a slice's histogram
constexpr double UNIT = 4398046511104.0;  // 2^42: a weight of 1

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab;
    int units, unit_blocks;  // blocks (16 bytes) of a unit, a multiple of 64
    int fine;                // groups of a unit whose maxima are kept: 64 lanes, or 4 rows of 16
    int cap;                 // entries a unit can list
    const float* u;
    const float* temperature_rows;
    const int32_t* top_k_rows;
    const float* top_p_rows;
    const float* min_p_rows;
    float temperature, top_p, min_p;
    int64_t top_k;
    int64_t* out_idx;
    float* out_logprob;
    // workspace
    double* unit_sum;      // [rows][units], of exp((l - unit's max) / temperature)
    float* unit_max;       // [rows][units]
    float* fine_max;       // [rows][units][fine]
    uint32_t* list_len;    // [rows][units]
    uint64_t* bin_amount;  // [rows][slices][BINS], of slices with long lists
    uint32_t* bin_count;   // [rows][slices][BINS]
    uint64_t* list;        // [rows][units][cap]
    __device__ __forceinline__ int slices() const { return (units + NW - 1) / NW; }
    // a slice lists entries only up to here without a histogram: all such together fit in LDS
    __device__ __forceinline__ uint32_t short_slice() const { return (uint32_t)(LIST / slices()); }
};

// One row's settings.
struct Setting {
    double c;  // log2(e) / temperature
    uint32_t k;
    double p, min_p;
    bool top_p_on, min_p_on;
    __device__ __forceinline__ Setting(const SampleArgs& a, int b)
    {
        const float t = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
        const int64_t kk = a.top_k_rows ? (int64_t)a.top_k_rows[b] : a.top_k;
        const float pp = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
        const float mm = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
        const bool greedy = !(t > 0.0f);
        c = greedy ? LOG2E_F64 : LOG2E_F64 / (double)fminf(t, FLT_MAX);
        k = greedy ? 1u : kk > 0 && kk < a.vocab ? (uint32_t)kk : 0u;
        top_p_on = pp < 1.0f;
        p = (double)fmaxf(pp, 0.0f);
        min_p_on = !(mm <= 0.0f);
        min_p = (double)fminf(mm, 1.0f);  // (NaN: 1)
    }
    __device__ __forceinline__ bool whole_sum() const { return k == 0 && (top_p_on || !min_p_on); }
    __device__ __forceinline__ bool listed() const { return k > 1 || (k == 0 && (top_p_on || min_p_on)); }
};

// A row in blocks of 16 bytes (the last possibly shorter), from its first
// column on: any alignment of the elements is taken, as the memory pipeline
// takes it.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

template <int LT>
struct Row {
    static constexpr int VEC = LT == VQ2_DT_F32 ? 4 : 8;
    const void* p;  // its first column
    int vocab, blocks;
    __device__ __forceinline__ Row(const SampleArgs& a, int b)
        : p((const char*)a.logits + b * a.stride * (16 / VEC)), vocab(a.vocab), blocks((a.vocab + VEC - 1) / VEC)
    {
    }
    __device__ __forceinline__ u32x4 raw(int block) const
    {
        if ((block + 1) * VEC <= vocab) return *(const u32x4_any*)((const char*)p + (int64_t)block * 16);
        // the last, short block, element by element
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = block * VEC + i * (VEC / 4);
            if constexpr (LT == VQ2_DT_F32) {
                w[i] = c < vocab ? ((const uint32_t*)p)[c] : 0xFF800000u;
            } else {
                constexpr uint32_t ABSENT = LT == VQ2_DT_F16 ? 0xFC00u : 0xFF80u;  // -inf
                w[i] = c < vocab ? ((const uint16_t*)p)[c] : ABSENT;
                w[i] |= (c + 1 < vocab ? ((const uint16_t*)p)[c + 1] : ABSENT) << 16;
            }
        }
        return w;
    }
    // An infinite logit becomes the largest finite one (no difference of
    // infinities); NaN stays.
    static __device__ __forceinline__ float finite(float v) { return v == INFINITY ? FLT_MAX : v; }
    static __device__ __forceinline__ void values(u32x4 w, float (&v)[VEC])
    {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            if constexpr (LT == VQ2_DT_F32) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const uint32_t h = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
                v[i] = LT == VQ2_DT_F16 ? f16_bits_to_f32((uint16_t)h) : bf16_bits_to_f32(h);
            }
            v[i] = finite(v[i]);
        }
    }
    __device__ __forceinline__ void load(int block, float (&v)[VEC]) const { values(raw(block), v); }
    __device__ __forceinline__ float at(int column) const { return finite(ld_t<LT>(p, column)); }
    // f(block, values) for the blocks from `from` on in steps of `step`, the
    // next block's load in flight meanwhile
    template <class F>
    __device__ __forceinline__ void stream(int from, int end, int step, F f) const
    {
        if (from >= end) return;
        u32x4 next = raw(from);
        for (int i = from; i < end; i += step) {
            const u32x4 w = next;
            if (i + step < end) next = raw(i + step);
            float v[VEC];
            values(w, v);
            f(i, v);
        }
    }
};

// Order of a row's entries: larger is earlier.
__device__ __forceinline__ uint64_t order_key(float l, int i)
{
    return argmax_key(l + 0.0f, i);  // (+ 0: -0 is 0)
}
__device__ __forceinline__ float key_logit(uint64_t key)
{
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ int key_column(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

__device__ __forceinline__ uint64_t fixed(double w) { return (uint64_t)(w * UNIT + 0.5); }

// A row's weights of 64 bits.
struct Weigher {
    float max;
    double c;
    __device__ __forceinline__ double operator()(float l) const
    {
        const double d = ((double)l - (double)max) * c;
        return d > -999.0 ? exp2_f64_in(d) : 0.0;  // (NaN: 0)
    }
};

// The bin of a logit, 0 the highest: linear between `max` and `max` - 1 / inv
// * BINS.  Rounded arithmetic, but monotonic: a higher logit is never in a
// lower bin.
__device__ __forceinline__ int bin_of(float l, float max, float inv)
{
    return (int)fminf((max - l) * inv, (float)(BINS - 1));
}
__device__ __forceinline__ float bins_inv(float max, float cut)
{
    const float width = max - cut;
    return width > 0.0f && width < INFINITY ? (float)BINS / width : 0.0f;
}

// ------------------------------------------------- sums over the workgroup
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

struct Scratch {
    uint64_t wave64[NW + 2];
    double wave_d[NW];
};

template <class T>
__device__ __forceinline__ T wave_scan(T v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const T o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// Inclusive running sum over the workgroup; total in every thread.
__device__ __forceinline__ uint64_t block_scan(Scratch& sh, uint64_t v, uint64_t& total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) sh.wave64[w] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const uint64_t x = sh.wave64[i];
        before += i < w ? x : 0;
        all += x;
    }
    total = all;
    return v + before;
}

// Largest value over the workgroup, in every thread.
__device__ __forceinline__ float block_max(Scratch& sh, float v)
{
    v = wave_max_all(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_d[threadIdx.x >> 6] = (double)v;
    __syncthreads();
    float m = (float)sh.wave_d[0];
#pragma unroll
    for (int i = 1; i < NW; i++) m = fmaxf(m, (float)sh.wave_d[i]);
    return m;
}

__device__ __forceinline__ uint64_t block_min(Scratch& sh, uint64_t v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t o = __shfl_xor(v, off);
        v = o < v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave64[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t m = sh.wave64[0];
#pragma unroll
    for (int i = 1; i < NW; i++) m = sh.wave64[i] < m ? sh.wave64[i] : m;
    return m;
}

// What the units say of a row: its maximum and, of a sum over the whole row, Z
// and each thread's running sum, thread t holding units 2 t and 2 t + 1.
struct Units {
    float um[2];
    float max;
    double us[2];  // weights relative to the row's maximum
    double z;
};

__device__ __forceinline__ Units read_units(Scratch& sh, const SampleArgs& a, const Setting& s, int b)
{
    Units r;
    const int64_t u0 = (int64_t)b * a.units;
    const int t = 2 * threadIdx.x;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        r.um[i] = t + i < a.units ? a.unit_max[u0 + t + i] : -INFINITY;
        r.us[i] = s.whole_sum() && t + i < a.units ? a.unit_sum[u0 + t + i] : 0.0;
    }
    r.max = block_max(sh, fmaxf(r.um[0], r.um[1]));
    r.z = 0.0;
    if (s.whole_sum()) {
#pragma unroll
        for (int i = 0; i < 2; i++) r.us[i] *= exp2_f64(((double)r.um[i] - (double)r.max) * s.c);
        const double w = wave_sum_f64(r.us[0] + r.us[1]);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.wave_d[threadIdx.x >> 6] = w;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) r.z += sh.wave_d[i];
    }
    return r;
}

// ------------------------------------------------------------------- stats
template <int LT>
__global__ void __launch_bounds__(NT) sample_stats_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    const int unit = blockIdx.x * NW + (threadIdx.x >> 6);
    if (unit >= a.units) return;
    const Setting s(a, b);
    const Row<LT> row(a, b);
    const int from = unit * a.unit_blocks + lane, end = min(row.blocks, (unit + 1) * a.unit_blocks);
    float m = -INFINITY;
    double sum = 0.0;
    if (s.whole_sum()) {
        // sum of exp((l - ref) / temperature), ref one of the lane's logits:
        // 64 bits hold weights of 2^1000, so it moves only where one is close
        float ref = -INFINITY;
        row.stream(from, end, 64, [&](int, const float (&v)[VEC]) {
            float top = v[0];
#pragma unroll
            for (int j = 1; j < VEC; j++) top = fmaxf(top, v[j]);
            m = fmaxf(m, top);
            if (((double)top - (double)ref) * s.c > 900.0) {
                sum *= exp2_f64(((double)ref - (double)top) * s.c);
                ref = top;
            }
#pragma unroll
            for (int j = 0; j < VEC; j++) sum += exp2_f64(((double)v[j] - (double)ref) * s.c);
        });
        const float um = wave_max_all(m);
        sum = wave_sum_f64(sum * exp2_f64(((double)ref - (double)um) * s.c));
    } else {
        row.stream(from, end, 64, [&](int, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++) m = fmaxf(m, v[j]);
        });
    }
    const int64_t at = (int64_t)b * a.units + unit;
    if (s.k > 1) {
        if (a.fine == 4) {
            float g = fmaxf(m, dpp_xor1(m));
            g = fmaxf(g, dpp_xor2(g));
            g = fmaxf(g, dpp_half_mirror(g));
            g = fmaxf(g, dpp_row_mirror(g));
            if ((lane & 15) == 0) a.fine_max[at * 4 + lane / 16] = g;
        } else {
            a.fine_max[at * 64 + lane] = m;
        }
    }
    m = wave_max_all(m);
    if (lane == 0) {
        a.unit_max[at] = m;
        a.unit_sum[at] = sum;
    }
}

// ----------------------------------------------------------------- collect
struct CollectShared {
    Scratch scratch;
    uint64_t amount[BINS];
    uint32_t count[NT];
    uint32_t slice_n;
};

// The logit from which on a row's entries may stay: rounded down, by more than
// the arithmetic here is off.
__device__ float lowest_kept(CollectShared& sh, const SampleArgs& a, const Setting& s, const Units& un, int b)
{
    const int tid = threadIdx.x;
    const double m = (double)un.max;
    double w = 2.8421709430404007e-14;  // 2^-45
    if (s.k == 0 && s.top_p_on) w = fmax(w, (1.0 - s.p) * 0.999 * un.z / (double)a.vocab);
    if (s.min_p_on && !(s.k > 0 && s.top_p_on)) w = fmax(w, s.min_p * 0.999);
    double low = m + log2(w) / s.c;
    if (s.k > 0) {
        // the lower end of the bin that the k-th largest maximum falls into;
        // more groups than k are needed for it to say something
        const bool coarse = s.k * 2 <= (uint32_t)a.units;
        const int groups = coarse ? a.units : a.units * a.fine;
        if (s.k * 5 <= (uint32_t)groups * 4) {
            const int64_t u0 = (int64_t)b * a.units;
            const float* const g = coarse ? a.unit_max + u0 : a.fine_max + u0 * a.fine;
            const float floor = (float)fmax(low, (double)-FLT_MAX);
            float least = INFINITY;
            for (int i = tid; i < groups; i += NT) least = fminf(least, fmaxf(g[i], floor));
            least = -block_max(sh.scratch, -least);
            const float width = un.max - least;
            const float inv = width > 0.0f && width < INFINITY ? (float)NT / width : 0.0f;
            auto bin = [&](float l) { return (int)fminf((un.max - l) * inv, (float)(NT - 1)); };
            sh.count[tid] = 0;
            __syncthreads();
            for (int i = tid; i < groups; i += NT) {
                const float l = g[i];
                if (l >= least) atomicAdd(&sh.count[bin(l)], 1u);
            }
            __syncthreads();
            uint64_t all;
            const uint64_t mine = sh.count[tid], run = block_scan(sh.scratch, mine, all);
            if (tid == 0) sh.scratch.wave64[NW] = NT;
            __syncthreads();
            if (run >= s.k && run - mine < s.k) sh.scratch.wave64[NW] = (uint64_t)tid;
            __syncthreads();
            const int r = (int)sh.scratch.wave64[NW];
            // the least maximum of the bins up to that one: k are at least as large
            float kth = INFINITY;
            if (r < NT)
                for (int i = tid; i < groups; i += NT) {
                    const float l = g[i];
                    if (l >= least && bin(l) <= r) kth = fminf(kth, l);
                }
            kth = -block_max(sh.scratch, -kth);
            if (r < NT) return fmaxf(kth, floor - (fabsf(floor) + fabsf(un.max)) * 1e-6f);
        }
    }
    const double slack = (fabs(m) + fabs(low)) * 1e-6;
    return (float)fmax(low - slack, (double)-FLT_MAX);
}

template <int LT>
__global__ void __launch_bounds__(NT) sample_collect_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ CollectShared sh;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const Setting s(a, b);
    if (!s.listed()) return;
    const Units un = read_units(sh.scratch, a, s, b);
    if (un.max == -INFINITY) return;
    const float cut = lowest_kept(sh, a, s, un, b);
    const Row<LT> row(a, b);
    const int64_t units0 = (int64_t)b * a.units;
    const int unit = blockIdx.x * NW + (tid >> 6);
    const int from = unit * a.unit_blocks, end = min(row.blocks, from + a.unit_blocks);
    if (tid == 0) sh.slice_n = 0;
    __syncthreads();
    if (unit < a.units) {
        uint64_t* const list = a.list + (units0 + unit) * a.cap;
        int n = 0;
        // (lanes past the end keep step, without entries)
        const int rounds = max(0, (end - from + 63) / 64);
        u32x4 next{};
        if (from + lane < end) next = row.raw(from + lane);
        for (int r = 0; r < rounds; r++) {
            const int i = from + r * 64 + lane;
            const u32x4 w = next;
            if (i + 64 < end) next = row.raw(i + 64);
            float v[VEC];
            Row<LT>::values(w, v);
            uint32_t in = 0;
#pragma unroll
            for (int j = 0; j < VEC; j++) in |= (uint32_t)(v[j] >= cut) << j;
            if (i >= end) in = 0;
            if (__ballot(in != 0) == 0) continue;
            const int mine = __popc(in), upto = wave_scan(mine);
            int at = n + upto - mine;
            if (in) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (in >> j & 1) {
                        if (at < a.cap) list[at] = order_key(v[j], i * VEC + j);
                        at++;
                    }
            }
            n += __shfl(upto, 63);
        }
        if (lane == 0) {
            a.list_len[units0 + unit] = (uint32_t)n;
            atomicAdd(&sh.slice_n, (uint32_t)n);
        }
    }
    __syncthreads();
    if (sh.slice_n <= a.short_slice()) return;
    // a histogram of the slice's entries beside their lists
    if (tid < BINS) {
        sh.amount[tid] = 0;
        sh.count[tid] = 0;
    }
    __syncthreads();
    const Weigher weigh{un.max, s.c};
    const float inv = bins_inv(un.max, cut);
    if (unit < a.units)
        row.stream(from + lane, end, 64, [&](int, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (v[j] >= cut) {
                    const int r = bin_of(v[j], un.max, inv);
                    atomicAdd((unsigned long long*)&sh.amount[r], (unsigned long long)fixed(weigh(v[j])));
                    atomicAdd(&sh.count[r], 1u);
                }
        });
    __syncthreads();
    if (tid < BINS) {
        const int64_t at = ((int64_t)b * gridDim.x + blockIdx.x) * BINS + tid;
        a.bin_amount[at] = sh.amount[tid];
        a.bin_count[at] = sh.count[tid];
    }
}

// ------------------------------------------------------------------ finish
struct FinishShared {
    Scratch scratch;
    CollectShared cut;        // (for lowest_kept)
    uint64_t list[LIST];      // the row's entries in column order
    uint64_t amount[NT];      // a histogram's sums; weights of ranked entries
    uint64_t small[NT];       // entries that are ranked
    uint32_t count[NT];
    uint32_t first[MAX_UNITS + 1];  // entries of the list before a unit's
    uint64_t slice_mass[MAX_SLICES];
    uint32_t small_n;
};

// The entries that a border is sought among: a list in LDS or, for a row whose
// ties fit none, every entry of the row from `cut` on.
template <int LT>
struct Source {
    const Row<LT>& row;
    const uint64_t* list;  // null: the row
    int n;
    float cut;
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        if (list) {
            for (int i = threadIdx.x; i < n; i += NT) f(list[i]);
        } else {
            row.stream(threadIdx.x, row.blocks, NT, [&](int i, const float (&v)[Row<LT>::VEC]) {
                for (int j = 0; j < Row<LT>::VEC; j++)
                    if (v[j] >= cut) f(order_key(v[j], i * Row<LT>::VEC + j));
            });
        }
    }
};

// The border of the entries in [lo, ~0]: the key of the last one that stays
// when an entry stays while the amounts before it are below `limit` (>= 1), of
// which `before` are ahead of them all.  Each round is a histogram of the
// keys over NT equal ranges, whose running sum finds the range that the limit
// falls into; keys differ, so ranges end up with few entries, which are
// ranked directly.  lo if all stay.
template <int LT, class F>
__device__ uint64_t find_border(FinishShared& sh, const Source<LT>& src, uint64_t lo, uint64_t limit, uint64_t before,
                                F amount)
{
    const int tid = threadIdx.x;
    uint64_t hi = 0;
    for (int round = 0;; round++) {
        // the range that the entries span
        uint64_t least = ~0ull, most = ~0ull;  // (most: the largest key's complement)
        src.each([&](uint64_t key) {
            if (key >= lo && (round == 0 || key <= hi)) {
                least = key < least ? key : least;
                most = ~key < most ? ~key : most;
            }
        });
        least = block_min(sh.scratch, least);
        most = ~block_min(sh.scratch, most);
        if (least == ~0ull) return lo;  // no entry
        lo = least;
        hi = most;
        const uint64_t span = hi - lo;
        constexpr int BITS = 9;
        static_assert(NT == 1 << BITS, "one range a thread");
        const int shift = span < NT ? 0 : 64 - __clzll(span) - BITS;
        __syncthreads();
        sh.amount[tid] = 0;
        sh.count[tid] = 0;
        __syncthreads();
        src.each([&](uint64_t key) {
            if (key >= lo && key <= hi) {
                const int r = (int)((hi - key) >> shift);
                atomicAdd((unsigned long long*)&sh.amount[r], (unsigned long long)amount(key));
                atomicAdd(&sh.count[r], 1u);
            }
        });
        __syncthreads();
        const uint64_t mine = sh.amount[tid];
        uint64_t all;
        const uint64_t run = before + block_scan(sh.scratch, mine, all);
        if (before + all < limit) return lo;
        if (run >= limit && run - mine < limit) {
            sh.scratch.wave64[NW] = (uint64_t)tid;
            sh.scratch.wave64[NW + 1] = run - mine;
        }
        __syncthreads();
        const int r = (int)(sh.scratch.wave64[NW] & (NT - 1));
        before = sh.scratch.wave64[NW + 1];
        const uint32_t m = min(sh.count[r], (uint32_t)NT);
        hi -= (uint64_t)r << shift;
        const uint64_t width = (1ull << shift) - 1;
        lo = hi - lo < width ? lo : hi - width;
        if (m > DIRECT && shift > 0) continue;
        if (tid == 0) sh.small_n = 0;
        __syncthreads();
        src.each([&](uint64_t key) {
            if (key >= lo && key <= hi) {
                const uint32_t at = atomicAdd(&sh.small_n, 1u) & (NT - 1);
                sh.small[at] = key;
                sh.amount[at] = amount(key);
            }
        });
        __syncthreads();
        uint64_t last = ~0ull;
        if (tid < (int)m) {
            const uint64_t key = sh.small[tid];
            uint64_t above = before;
            for (int j = 0; j < (int)m; j++) above += sh.small[j] > key ? sh.amount[j] : 0;
            if (above < limit) last = key;
        }
        return block_min(sh.scratch, last);
    }
}

__device__ __forceinline__ double clamped_u(const SampleArgs& a, int b) { return fmin(fmax((double)a.u[b], 0.0), 1.0); }

__device__ __forceinline__ void write_token(const SampleArgs& a, int b, int column, float l, const Weigher& weigh,
                                            double total)
{
    a.out_idx[b] = column;
    a.out_logprob[b] = (float)(((double)l - (double)weigh.max) * weigh.c / LOG2E_F64 - log(total));
}

// The token at `target` of the kept entries of the list in column order; its
// entries' kept weights are `kept`, `total` all of them.
template <class F>
__device__ void draw_from_list(Scratch& sh, const SampleArgs& a, const Weigher& weigh, const uint64_t* list, int n, F kept,
                               uint64_t target, uint64_t total, int b)
{
    const int per = (n + NT - 1) / NT, i0 = threadIdx.x * per, i1 = min(n, i0 + per);
    uint64_t mine = 0, all;
    for (int i = i0; i < i1; i++) mine += kept(list[i]);
    uint64_t run = block_scan(sh, mine, all);
    if (!(run > target && run - mine <= target)) return;
    run -= mine;
    for (int i = i0; i < i1; i++) {
        run += kept(list[i]);
        if (run > target) {
            write_token(a, b, key_column(list[i]), key_logit(list[i]), weigh, (double)total / UNIT);
            return;
        }
    }
}

__device__ __forceinline__ uint64_t draw_target(const SampleArgs& a, int b, uint64_t total)
{
    const uint64_t t = (uint64_t)(clamped_u(a, b) * (double)total);
    return t < total ? t : total - 1;
}

// Up to DIRECT entries: each one's rank and the weight before it by comparing
// it with every other, half of them by each half of the workgroup.
__device__ void finish_direct(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh, int n, double z,
                              int b)
{
    static_assert(NT == 2 * DIRECT, "two threads an entry");
    const int tid = threadIdx.x, i = tid & (DIRECT - 1), half = tid / DIRECT;
    const uint64_t key = i < n ? sh.list[i] : 0;
    const double w = weigh(key_logit(key));
    const uint64_t mass = i < n ? fixed(w) : 0;
    if (half == 0) sh.amount[i] = mass;
    __syncthreads();
    uint32_t rank = 0;
    uint64_t before = 0;
    if (i < n) {
        const int mid = n / 2;
        for (int j = half ? mid : 0; j < (half ? n : mid); j++) {
            const bool ahead = sh.list[j] > key;
            rank += ahead;
            before += ahead ? sh.amount[j] : 0;
        }
    }
    sh.small[tid] = before;
    sh.count[tid] = rank;
    __syncthreads();
    rank += sh.count[tid ^ DIRECT];
    before += sh.small[tid ^ DIRECT];
    bool stays = half == 0 && i < n && (s.k == 0 || rank < s.k);
    uint64_t total;
    if (s.top_p_on) {
        double all = z * UNIT;
        if (s.k > 0) {
            block_scan(sh.scratch, stays ? mass : 0, total);
            all = (double)total;
        }
        stays = stays && (rank == 0 || (double)before < s.p * all);
    }
    if (s.min_p_on) stays = stays && w >= s.min_p;
    const uint64_t mine = stays ? mass : 0;
    const uint64_t run = block_scan(sh.scratch, mine, total);
    const uint64_t target = draw_target(a, b, total);
    if (run > target && run - mine <= target)
        write_token(a, b, key_column(key), key_logit(key), weigh, (double)total / UNIT);
}

// The row, all of it, by its source: borders by find_border, the draw from
// the list or, without one, over the row in pieces of the threads.
template <int LT>
__device__ void finish_source(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh,
                              const Source<LT>& src, double z, int b)
{
    auto mass = [&](uint64_t key) { return fixed(weigh(key_logit(key))); };
    uint64_t lo = 0, total;
    if (s.k > 0) lo = find_border(sh, src, lo, (uint64_t)s.k, 0, [](uint64_t) { return 1ull; });
    if (s.top_p_on) {
        double all = z * UNIT;
        if (s.k > 0) {
            uint64_t part = 0;
            src.each([&](uint64_t key) { part += key >= lo ? mass(key) : 0; });
            block_scan(sh.scratch, part, total);
            all = (double)total;
        }
        const double limit = ceil(s.p * all);
        lo = find_border(sh, src, lo, limit > 1.0 ? (uint64_t)limit : 1, 0, mass);
    }
    auto kept = [&](uint64_t key) -> uint64_t {
        if (key < lo) return 0;
        const double w = weigh(key_logit(key));
        return !s.min_p_on || w >= s.min_p ? fixed(w) : 0;
    };
    if (src.list) {
        uint64_t part = 0;
        src.each([&](uint64_t key) { part += kept(key); });
        block_scan(sh.scratch, part, total);
        draw_from_list(sh.scratch, a, weigh, src.list, src.n, kept, draw_target(a, b, total), total, b);
        return;
    }
    const int per = (a.vocab + NT - 1) / NT, c0 = threadIdx.x * per, c1 = min(a.vocab, c0 + per);
    auto at = [&](int c) -> uint64_t {
        const float l = src.row.at(c);
        return l >= src.cut ? kept(order_key(l, c)) : 0;
    };
    uint64_t mine = 0;
    for (int c = c0; c < c1; c++) mine += at(c);
    uint64_t run = block_scan(sh.scratch, mine, total);
    const uint64_t target = draw_target(a, b, total);
    if (!(run > target && run - mine <= target)) return;
    run -= mine;
    for (int c = c0; c < c1; c++) {
        run += at(c);
        if (run > target) {
            write_token(a, b, c, src.row.at(c), weigh, (double)total / UNIT);
            return;
        }
    }
}

// The smallest key whose weight is at least min_p, by a search of 64 steps at
// once in every wave.
__device__ __forceinline__ uint64_t min_p_border(const Setting& s, const Weigher& weigh)
{
    uint32_t lo = 0x00800000u, hi = (uint32_t)(order_key(weigh.max, 0) >> 32);  // (-FLT_MAX's; weight 1 >= min_p)
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, probe = lo + min((threadIdx.x & 63) * step, hi - lo);
        const uint64_t yes = __ballot(weigh(key_logit((uint64_t)probe << 32)) >= s.min_p);
        if (yes == 0) {
            lo = lo + min(63 * step, hi - lo - 1) + 1;
        } else {
            const int f = __ffsll((unsigned long long)yes) - 1;
            hi = lo + min((uint32_t)f * step, hi - lo);
            if (f > 0) lo = lo + min((uint32_t)(f - 1) * step, hi - lo) + (hi > lo ? 1 : 0);
            lo = min(lo, hi);
        }
    }
    return (uint64_t)hi << 32;
}

// A row of more entries than LDS lists: slices above short_slice() entries
// have histograms, the others' lists are in LDS.  False if a border's bin has
// too many entries.
template <int LT>
__device__ bool finish_long(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh, const Row<LT>& row,
                            float cut, double z, const uint64_t long_slices[MAX_SLICES / 64], int n, int b)
{
    constexpr int VEC = Row<LT>::VEC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slices = a.slices();
    const int64_t hist0 = (int64_t)b * slices * BINS;
    const int slice_blocks = NW * a.unit_blocks;
    const float inv = bins_inv(weigh.max, cut);
    auto mass = [&](uint64_t key) { return fixed(weigh(key_logit(key))); };
    auto is_long = [&](int g) { return (long_slices[g / 64] >> (g & 63) & 1) != 0; };
    // the row's histogram: two threads a bin, then the short slices' entries
    uint64_t* const amount = sh.amount;
    uint32_t* const count = sh.count;
    __syncthreads();
    amount[tid] = 0;
    count[tid] = 0;
    __syncthreads();
    {
        uint64_t am = 0;
        uint32_t ct = 0;
        for (int g = tid / BINS; g < slices; g += NT / BINS)
            if (is_long(g)) {
                am += a.bin_amount[hist0 + g * BINS + tid % BINS];
                ct += a.bin_count[hist0 + g * BINS + tid % BINS];
            }
        atomicAdd((unsigned long long*)&amount[tid % BINS], (unsigned long long)am);
        atomicAdd(&count[tid % BINS], ct);
        for (int i = tid; i < n; i += NT) {
            const uint64_t key = sh.list[i];
            const int r = bin_of(key_logit(key), weigh.max, inv);
            atomicAdd((unsigned long long*)&amount[r], (unsigned long long)mass(key));
            atomicAdd(&count[r], 1u);
        }
    }
    __syncthreads();
    const uint64_t bin_mass = tid < BINS ? amount[tid] : 0, bin_n = tid < BINS ? count[tid] : 0;
    // entries of bin r of all slices to sh.small, in any order; false if too many
    auto fetch = [&](int r) -> bool {
        if (tid == 0) sh.small_n = 0;
        __syncthreads();
        auto take = [&](uint64_t key) {
            const uint32_t at = atomicAdd(&sh.small_n, 1u);
            if (at < NT) sh.small[at] = key;
        };
        for (int g = wave; g < slices; g += NW) {
            if (!is_long(g)) continue;
            row.stream(g * slice_blocks + lane, min(row.blocks, (g + 1) * slice_blocks), 64, [&](int i, const float (&v)[VEC]) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (v[j] >= cut && bin_of(v[j], weigh.max, inv) == r) take(order_key(v[j], i * VEC + j));
            });
        }
        for (int i = tid; i < n; i += NT)
            if (bin_of(key_logit(sh.list[i]), weigh.max, inv) == r) take(sh.list[i]);
        __syncthreads();
        return sh.small_n <= NT;
    };
    // the border of `limit` by the bins' amounts `mine`: its bin, then among the bin's entries from `from` on
    int lo_bin = BINS;
    auto border = [&](uint64_t mine, uint64_t limit, uint64_t from, uint64_t& lo, auto per_entry) -> bool {
        uint64_t all;
        const uint64_t run = block_scan(sh.scratch, mine, all);
        if (all < limit) return true;
        if (run >= limit && run - mine < limit) {
            sh.scratch.wave64[NW] = (uint64_t)tid;
            sh.scratch.wave64[NW + 1] = run - mine;
        }
        __syncthreads();
        const int r = (int)(sh.scratch.wave64[NW] & (BINS - 1));
        const uint64_t before = sh.scratch.wave64[NW + 1];
        __syncthreads();
        if (!fetch(r)) return false;
        const int m = (int)sh.small_n;
        uint64_t last = ~0ull;
        if (tid < m && sh.small[tid] >= from) {
            const uint64_t key = sh.small[tid];
            uint64_t above = before;
            for (int j = 0; j < m; j++) above += sh.small[j] > key ? per_entry(sh.small[j]) : 0;
            if (above < limit) last = key;
        }
        last = block_min(sh.scratch, last);
        lo = last > lo && last != ~0ull ? last : lo;
        lo_bin = r;
        return true;
    };
    uint64_t lo = 0, total;
    double all_mass = z * UNIT;
    if (s.k > 0) {
        if (!border(bin_n, (uint64_t)s.k, 0, lo, [](uint64_t) { return 1ull; })) return false;
        if (s.top_p_on) {  // what top-k kept: whole bins, and the border's bin's entries
            uint64_t part = tid < lo_bin ? bin_mass : 0;
            if (lo_bin < BINS && tid < (int)sh.small_n && sh.small[tid] >= lo) part += mass(sh.small[tid]);
            block_scan(sh.scratch, part, total);
            all_mass = (double)total;
        }
    }
    if (s.top_p_on) {
        const double limit = ceil(s.p * all_mass);
        if (!border(bin_mass, limit > 1.0 ? (uint64_t)limit : 1, lo, lo, mass)) return false;
    }
    if (s.min_p_on) {
        const uint64_t at = min_p_border(s, weigh);
        if (at > lo) {
            lo = at;
            lo_bin = bin_of(key_logit(at), weigh.max, inv);
            __syncthreads();
            if (!fetch(lo_bin)) return false;
        }
    }
    // each slice's kept weight: its bins above the border's, its entries in that bin
    for (int g = tid; g < MAX_SLICES; g += NT) sh.slice_mass[g] = 0;
    __syncthreads();
    for (int g = wave; g < slices; g += NW) {
        if (!is_long(g)) continue;
        uint64_t part = 0;
        for (int r = lane; r < min(lo_bin, BINS); r += 64) part += a.bin_amount[hist0 + g * BINS + r];
        if (part) atomicAdd((unsigned long long*)&sh.slice_mass[g], (unsigned long long)part);
    }
    auto slice_of = [&](uint64_t key) { return key_column(key) / (slice_blocks * VEC); };
    if (lo_bin < BINS && tid < (int)sh.small_n) {
        const uint64_t key = sh.small[tid];
        if (key >= lo && is_long(slice_of(key)))
            atomicAdd((unsigned long long*)&sh.slice_mass[slice_of(key)], (unsigned long long)mass(key));
    }
    for (int i = tid; i < n; i += NT) {
        const uint64_t key = sh.list[i];
        if (key >= lo) atomicAdd((unsigned long long*)&sh.slice_mass[slice_of(key)], (unsigned long long)mass(key));
    }
    __syncthreads();
    const uint64_t mine = tid < slices ? sh.slice_mass[tid] : 0;
    const uint64_t run = block_scan(sh.scratch, mine, total);
    uint64_t target = draw_target(a, b, total);
    if (run > target && run - mine <= target) {
        sh.scratch.wave64[NW] = (uint64_t)tid;
        sh.scratch.wave64[NW + 1] = run - mine;
    }
    __syncthreads();
    const int g = (int)(sh.scratch.wave64[NW] & (MAX_SLICES - 1));
    target -= sh.scratch.wave64[NW + 1];
    auto kept = [&](uint64_t key) -> uint64_t { return key >= lo && slice_of(key) == g ? mass(key) : 0; };
    if (!is_long(g)) {
        draw_from_list(sh.scratch, a, weigh, sh.list, n, kept, target, total, b);
        return true;
    }
    const int b0 = g * slice_blocks, per = (slice_blocks + NT - 1) / NT;
    const int i0 = b0 + tid * per, i1 = min(min(row.blocks, b0 + slice_blocks), i0 + per);
    uint64_t part = 0, all;
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (v[j] >= cut) part += kept(order_key(v[j], i * VEC + j));
    });
    uint64_t upto = block_scan(sh.scratch, part, all);
    if (!(upto > target && upto - part <= target)) return true;
    upto -= part;
    for (int c = i0 * VEC; c < min(a.vocab, i1 * VEC); c++) {
        const float l = row.at(c);
        if (l >= cut) upto += kept(order_key(l, c));
        if (upto > target) {
            write_token(a, b, c, l, weigh, (double)total / UNIT);
            return true;
        }
    }
    return true;
}

// A draw over the whole row: the unit, then the column, whose running sum is
// the first above u Z (the last with a weight, if rounding leaves none).
template <int LT>
__device__ void finish_plain(FinishShared& sh, const SampleArgs& a, const Weigher& weigh, const Row<LT>& row, const Units& un,
                             int b)
{
    constexpr int VEC = Row<LT>::VEC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double* const ends = (double*)sh.amount;  // each thread's running sum
    // the thread at whose end the running sum of `mine` first exceeds target, and the sum before it
    auto locate = [&](double mine, double base, double target, double& before) -> int {
        const double run = wave_scan(mine);
        __syncthreads();
        if (lane == 63) sh.scratch.wave_d[wave] = run;
        __syncthreads();
        double at = base;
        for (int i = 0; i < wave; i++) at += sh.scratch.wave_d[i];
        ends[tid] = at + run;
        uint64_t t = block_min(sh.scratch, mine > 0.0 && at + run > target ? tid : NT);
        if (t == NT) t = NT - 1 - block_min(sh.scratch, mine > 0.0 ? NT - 1 - tid : NT - 1);
        before = t ? ends[t - 1] : base;
        return (int)t;
    };
    const double target = clamped_u(a, b) * un.z;
    double before;
    const int t = locate(un.us[0] + un.us[1], 0.0, target, before);
    // of that thread's two units
    if (tid == t) {
        const bool second = !(un.us[0] > 0.0) || (un.us[1] > 0.0 && !(before + un.us[0] > target));
        sh.scratch.wave64[NW] = (uint64_t)(2 * t + second);
        sh.slice_mass[0] = __builtin_bit_cast(uint64_t, second ? before + un.us[0] : before);
    }
    __syncthreads();
    const int unit = (int)sh.scratch.wave64[NW];
    const double base = __builtin_bit_cast(double, sh.slice_mass[0]);
    const int b0 = unit * a.unit_blocks, per = (a.unit_blocks + NT - 1) / NT;
    const int i0 = b0 + tid * per, i1 = min(min(row.blocks, b0 + a.unit_blocks), i0 + per);
    double mine = 0.0;
    row.stream(i0, i1, 1, [&](int, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++) mine += weigh(v[j]);
    });
    if (tid != locate(mine, base, target, before)) return;
    int col = -1;
    float l = weigh.max;
    for (int c = i0 * VEC; c < min(a.vocab, i1 * VEC) && (col < 0 || !(before > target)); c++) {
        const float v = row.at(c);
        const double w = weigh(v);
        before += w;
        if (w > 0.0) {
            col = c;
            l = v;
        }
    }
    write_token(a, b, col, l, weigh, un.z);
}

template <int LT>
__global__ void __launch_bounds__(NT) sample_finish_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ FinishShared sh;
    const int b = blockIdx.x, tid = threadIdx.x;
    const Setting s(a, b);
    const Row<LT> row(a, b);
    const int64_t units0 = (int64_t)b * a.units;
    const Units un = read_units(sh.scratch, a, s, b);
    if (un.max == -INFINITY) {
        if (tid == 0) {
            a.out_idx[b] = -1;
            a.out_logprob[b] = NAN;
        }
        return;
    }
    const Weigher weigh{un.max, s.c};
    if (s.k == 1) {  // the first maximum
        const int mine = un.um[0] == un.max ? 2 * tid : un.um[1] == un.max ? 2 * tid + 1 : MAX_UNITS;
        const int unit = (int)block_min(sh.scratch, (uint64_t)mine);
        uint64_t col = ~0ull;
        row.stream(unit * a.unit_blocks + tid, min(row.blocks, (unit + 1) * a.unit_blocks), NT,
                   [&](int i, const float (&v)[VEC]) {
#pragma unroll
                       for (int j = VEC - 1; j >= 0; j--)
                           if (v[j] == un.max && (uint64_t)(i * VEC + j) < col) col = (uint64_t)(i * VEC + j);
                   });
        col = block_min(sh.scratch, col);
        if (tid == 0) {
            a.out_idx[b] = (int64_t)col;
            a.out_logprob[b] = 0.0f;
        }
        return;
    }
    if (!s.listed()) {
        finish_plain<LT>(sh, a, weigh, row, un, b);
        return;
    }
    // the units' lists: all of them, or those of the slices without a histogram
    uint32_t len[2];
    bool over = false;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        len[i] = 2 * tid + i < a.units ? a.list_len[units0 + 2 * tid + i] : 0;
        over |= len[i] > (uint32_t)a.cap;
    }
    uint64_t all;
    block_scan(sh.scratch, (uint64_t)(len[0] + len[1]) | (over ? 1ull << 40 : 0), all);
    const bool fits = all <= LIST;
    uint64_t long_slices[MAX_SLICES / 64] = {};
    if (!fits) {
        // a slice's entries are those of the threads of its 8 units, 4 lanes
        uint32_t n = len[0] + len[1];
        n += __shfl_xor(n, 1);
        n += __shfl_xor(n, 2);
        const bool is_long = n > a.short_slice();
        if (is_long) len[0] = len[1] = 0;
        const uint64_t quads = __ballot(is_long && (tid & 3) == 0);
        __syncthreads();
        if ((tid & 63) == 0) {
            uint32_t bits = 0;
            for (int i = 0; i < 16; i++) bits |= (uint32_t)(quads >> (4 * i) & 1) << i;
            sh.scratch.wave64[tid >> 6] = bits;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) long_slices[i / 4] |= sh.scratch.wave64[i] << (16 * (i % 4));
    }
    const uint64_t upto = block_scan(sh.scratch, len[0] + len[1], all);
    const int n = (int)all;
    sh.first[2 * tid + 2] = (uint32_t)upto;
    sh.first[2 * tid + 1] = (uint32_t)upto - len[1];
    if (tid == 0) sh.first[0] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
        int at = 0;  // the unit: first[at] <= i < first[at + 1]
#pragma unroll
        for (int step = MAX_UNITS / 2; step > 0; step >>= 1)
            if (sh.first[at + step] <= (uint32_t)i) at += step;
        sh.list[i] = a.list[(units0 + at) * a.cap + (i - sh.first[at])];
    }
    __syncthreads();
    if (fits && n <= DIRECT) {
        finish_direct(sh, a, s, weigh, n, un.z, b);
        return;
    }
    float cut = -INFINITY;
    if (!fits) {
        cut = lowest_kept(sh.cut, a, s, un, b);
        if (finish_long<LT>(sh, a, s, weigh, row, cut, un.z, long_slices, n, b)) return;
        __syncthreads();
    }
    finish_source<LT>(sh, a, s, weigh, Source<LT>{row, fits ? sh.list : nullptr, n, cut}, un.z, b);
}

// How a call is cut: units of at least 64 blocks (one load a lane), longer
// ones where the rows alone make 1024 workgroups of 16 units.
struct Plan {
    int units, unit_blocks, fine, cap;
    size_t unit_sum, unit_max, fine_max, list_len, bin_amount, bin_count, list, bytes;
};

Plan make_plan(int64_t rows, int64_t vocab, int vec)
{
    Plan p;
    const int64_t blocks = (vocab + vec - 1) / vec;
    int64_t per = (blocks * rows + 16383) / 16384;
    per = per > (blocks + MAX_UNITS - 1) / MAX_UNITS ? per : (blocks + MAX_UNITS - 1) / MAX_UNITS;
    per = per > (blocks + NW - 1) / NW ? (blocks + NW - 1) / NW : per;
    p.unit_blocks = (int)((per + 63) / 64 * 64);
    p.units = (int)((blocks + p.unit_blocks - 1) / p.unit_blocks);
    p.fine = p.units >= 512 ? 4 : 64;
    const int entries = p.unit_blocks * vec;
    // a list of more is not read: its slice has a histogram (short_slice())
    const int whole = LIST / ((p.units + NW - 1) / NW) > 512 ? LIST / ((p.units + NW - 1) / NW) : 512;
    p.cap = entries < whole ? entries : whole;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t r = at;
        at += (n + 255) / 256 * 256;
        return r;
    };
    const size_t n = (size_t)rows * p.units, slices = (size_t)rows * ((p.units + NW - 1) / NW);
    p.unit_sum = take(n * 8);
    p.unit_max = take(n * 4);
    p.fine_max = take(n * p.fine * 4);
    p.list_len = take(n * 4);
    p.bin_amount = take(slices * BINS * 8);
    p.bin_count = take(slices * BINS * 4);
    p.list = take(n * p.cap * 8);
    p.bytes = at;
    return p;
}

template <int LT>
int launch(const SampleCall& c)
{
    const Plan p = make_plan(c.rows, c.vocab, Row<LT>::VEC);
    char* const ws = (char*)c.workspace;
    const SampleArgs a{c.logits, c.l_stride, (int)c.vocab, p.units, p.unit_blocks, p.fine, p.cap,
                       c.u, c.temperature_rows, c.top_k_rows, c.top_p_rows, c.min_p_rows,
                       c.temperature, c.top_p, c.min_p, c.top_k, c.out_idx, c.out_logprob,
                       (double*)(ws + p.unit_sum), (float*)(ws + p.unit_max), (float*)(ws + p.fine_max),
                       (uint32_t*)(ws + p.list_len), (uint64_t*)(ws + p.bin_amount), (uint32_t*)(ws + p.bin_count),
                       (uint64_t*)(ws + p.list)};
    // nothing is listed for settings, common to all rows, without a border
    const bool listed = c.temperature_rows || c.top_k_rows || c.top_p_rows || c.min_p_rows ||
                        (c.temperature > 0.0f && c.top_k != 1 && (c.top_k > 0 || c.top_p < 1.0f || c.min_p > 0.0f));
    hipStream_t st = (hipStream_t)c.stream;
    const dim3 grid((unsigned)((p.units + NW - 1) / NW), (unsigned)c.rows), block(NT);
    hipLaunchKernelGGL(sample_stats_kernel<LT>, grid, block, 0, st, a);
    if (listed) hipLaunchKernelGGL(sample_collect_kernel<LT>, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_finish_kernel<LT>, dim3((unsigned)c.rows), block, 0, st, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_hip_error(err, "vq2 sample launch");
    return VQ2_OK;
}

}  // namespace

size_t sample_workspace_bytes(int64_t rows, int64_t vocab)
{
    if (rows < 1 || rows > VQ2_SAMPLE_MAX_ROWS || vocab < 1 || vocab > VQ2_SAMPLE_MAX_VOCAB) return 0;
    const size_t f32 = make_plan(rows, vocab, 4).bytes, f16 = make_plan(rows, vocab, 8).bytes;
    return f32 > f16 ? f32 : f16;
}

int sample_launch(const SampleCall& c)
{
    if (c.l_dt == VQ2_DT_F32) return launch<VQ2_DT_F32>(c);
    if (c.l_dt == VQ2_DT_F16) return launch<VQ2_DT_F16>(c);
    return launch<VQ2_DT_BF16>(c);
}

}  // namespace vq2
