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
// draw in some hundred would be another.  So weights are computed in 64 bits,
// and where entries are put in order they are summed as whole numbers of 2^-42
// of the largest (a weight below 2^-43 counts as 0), whose sum is the same in
// any order.
//
// Launches:
//   stats    A row is cut into units, each a contiguous piece that one wave
//            reads; every unit's maximum and weight (for top-k, the maxima of
//            finer groups).
//   collect  The row's maximum and total are known from the units and with
//            them a logit below which nothing can stay:
//              top-k  the k-th largest of the groups' maxima (k entries are
//                     that large);
//              top-p  w < (1 - p) Z / V: all such entries together weigh less
//                     than (1 - p) Z, which the last entries may be short of;
//              min-p  the least logit of w >= min_p;  always: w < 2^-45.
//            The entries above, usually some hundred to some thousand of a
//            row, go to the row's list, in any order.
//   refine   Only for rows with more entries than LDS holds (flat rows): their
//            slices (the units of a workgroup) left histograms; each workgroup
//            adds them up to the bin that the border lies in, and lists its
//            slice's entries of that bin.
//   finish   One workgroup a row, on the list in LDS: up to 128 entries are
//            ranked directly, more are narrowed down by a histogram (in the
//            order of logits for a border, of columns for the draw).
// A draw without a border (no top-k, top-p or min-p) is stats and finish: the
// unit whose weights' running sum passes u Z is read again.
//
// Kernel times on MI355X, us (stats + collect + refine + finish):
//   1 x 151936 fp32, top-k 50, top-p 0.9     3.2 + 7.0 +  -  +  5.3
//   1 x 151936 fp32, top-p 0.95              4.1 + 6.0 + 1.9 +  8.8
//   8 x 32000 fp16, top-k 1000               4.0 + 7.9 + 1.9 + 12.5
//   37 x 50257 bf16, settings by row         5.9 + 9.5 + 6.7 + 13.3
//   256 x 151936 fp32, plain                  36 +  -  +  -  + 10.2
//   256 x 151936 bf16, top-p 0.9, min-p       29 +  17 + 4.6 +  7.2
// Small calls are chains of launches and, within them, of loads and barriers of
// one row.  In large ones the stats launch is most.  Over fp32 it reads 4.3 TB/s
// (a large copy reaches 4.9; with the exponentials left out, 29 us).  Over 16
// bits vector instructions bound it: 21 a logit, issuing in 92 % of the busy
// cycles (76 % over fp32); the table's lookups conflict in 20 % of them, hidden.
// A row whose border lies among more entries than the list holds is gone over by
// one workgroup, bound by that compute unit's instructions.  Those are rows flat
// to a tenth, long ties, and rows whose top-p border is far down their tail (0.98
// of a power law at a temperature of 1.15, 126731 entries of bf16 above the
// border, 4000 in its bin): 0.25 to 0.33 ms at 151936 logits, 0.48 with ties of
// which every second column is one, 0.47 to 0.7 ms where it has both a longer
// top-k and a top-p.
#include <float.h>

#include "vq2_common.hpp"
#include "vq2_router.hpp"
#include "vq2_internal.hpp"

namespace vq2 {

namespace {

constexpr int NT = 512;           // threads of a workgroup
constexpr int BITS = 9;           // NT = 2^BITS
constexpr int NW = NT / 64;       // its waves, one unit each: a slice
constexpr int MAX_UNITS = 1024;   // units of a row
constexpr int MAX_GROUPS = 8192;  // groups of a row (Plan::fine)
constexpr int LIST = 2944;        // entries of the list in LDS
constexpr int SHORT_LIST = 8192;  // entries of the slices without a histogram
constexpr int DIRECT = 128;       // entries that are ranked directly
constexpr int PARTS = NT / DIRECT;  // threads an entry then
constexpr int BINS = 256;         // of a slice's histogram
constexpr double UNIT = 4398046511104.0;  // 2^42: a weight of 1
static_assert(NT == 1 << BITS && NT >= MAX_UNITS / 2, "a thread a range and for two units");

// What the collect launch leaves of a row.
struct RowInfo {
    double z;
    float max, cut;
};
// What the refine launch leaves: the border's bin and the amount ahead of it.
struct RefineInfo {
    uint64_t before;
    int64_t bin;  // -1: all entries stay
};
enum { CNT_LONG, CNT_SHORT, CNT_BIN, CNTS };  // a row's counters

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab;
    int units, unit_blocks;  // blocks (16 bytes) of a unit, a multiple of 64
    int fine;                // groups of a unit whose maxima are kept: 64 lanes, or their quads or rows of 16
    int list_cap, short_cap; // entries of the lists
    bool refines;            // the refine launch takes place
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
    uint32_t* counters;    // [rows][CNTS]
    RowInfo* info;         // [rows]
    RefineInfo* refined;   // [rows]
    uint32_t* slice_n;     // [rows][slices] entries
    uint64_t* slice_mass;  // [rows][slices] of the bins ahead of the border's
    uint64_t* bin_amount;  // [rows][slices][BINS], of slices of more than short_slice() entries
    uint32_t* bin_count;   // [rows][slices][BINS]
    uint64_t* list;        // [rows][list_cap] entries of such slices; then of the border's bin
    uint64_t* short_list;  // [rows][short_cap] entries of the others
    __device__ __forceinline__ int slices() const { return (units + NW - 1) / NW; }
    // all slices of up to so many entries together fit the short list (and one a stage)
    __device__ __forceinline__ uint32_t short_slice() const { return (uint32_t)min(short_cap / slices(), LIST); }
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
        k = greedy || kk == 1 ? 1u : kk > 0 && kk < a.vocab ? (uint32_t)kk : 0u;  // (1 also of one column, as launch() has it)
        top_p_on = pp < 1.0f;
        p = (double)fmaxf(pp, 0.0f);
        min_p_on = !(mm <= 0.0f);
        min_p = (double)fminf(mm, 1.0f);  // (NaN: 1)
    }
    __device__ __forceinline__ bool whole_sum() const { return k == 0 && (top_p_on || !min_p_on); }
    __device__ __forceinline__ bool listed() const { return k > 1 || (k == 0 && (top_p_on || min_p_on)); }
    // one border is enough to say what stays (besides the collect's cut)
    __device__ __forceinline__ bool one_border() const { return k == 0 || !top_p_on; }
};

// A row in blocks of 16 bytes from its first column on, whatever the
// alignment of its elements; the last block may be short.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

// An infinite logit as the largest finite one, for what takes no infinity; NaN
// stays.
__device__ __forceinline__ float finite(float v) { return v == INFINITY ? FLT_MAX : v; }

template <int LT>
struct Row {
    static constexpr int VEC = LT == VQ2_DT_F32 ? 4 : 8;
    const char* p;  // its first column
    int vocab, blocks, full;
    __device__ __forceinline__ Row(const SampleArgs& a, int b)
        : p((const char*)a.logits + b * a.stride * (16 / VEC)), vocab(a.vocab), blocks((a.vocab + VEC - 1) / VEC),
          full(a.vocab / VEC)
    {
    }
    __device__ __forceinline__ u32x4 raw(int block) const { return *(const u32x4_any*)(p + (int64_t)block * 16); }
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
        }
    }
    // f(block, values) for the blocks from `from` on in steps of `step`, the
    // next block's load in flight meanwhile; the first one's is head(from,
    // end).  A short last block is loaded by itself and padded with -inf.
    __device__ __forceinline__ u32x4 head(int from, int end) const
    {
        return from < min(end, full) ? raw(from) : u32x4{};
    }
    template <class F>
    __device__ __forceinline__ void stream(int from, int end, int step, F f) const
    {
        stream(from, end, step, head(from, end), f);
    }
    template <class F>
    __device__ __forceinline__ void stream(int from, int end, int step, u32x4 next, F f) const
    {
        for (int i = from; i < end; i += step) {
            const u32x4 w = next;
            if (i + step < min(end, full)) next = raw(i + step);
            float v[VEC];
            values(w, v);
            if (i >= full) {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[j] = i * VEC + j < vocab ? ld_t<LT>(p, i * VEC + j) : -INFINITY;
            }
            f(i, v);
        }
    }
    // the same with 16 values a thread in flight
    template <class F>
    __device__ __forceinline__ void stream_wide(int from, int end, int step, F f) const
    {
        constexpr int Q = 16 / VEC;
        int i = from;
        for (; i + (Q - 1) * step < min(end, full); i += Q * step) {
            u32x4 w[Q];
#pragma unroll
            for (int q = 0; q < Q; q++) w[q] = raw(i + q * step);
#pragma unroll
            for (int q = 0; q < Q; q++) {
                float v[VEC];
                values(w[q], v);
                f(i + q * step, v);
            }
        }
        stream(i, end, step, f);
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

// A row's weights of 64 bits.  The maximum weighs 1, also an infinite one (no
// difference of infinities), beside which every finite logit weighs nothing.
struct Weigher {
    float max;
    double c;
    // log2 of the weight
    __device__ __forceinline__ double log2_of(float l) const { return l == max ? 0.0 : ((double)l - (double)max) * c; }
    __device__ __forceinline__ double operator()(float l) const
    {
        const double d = log2_of(l);
        return d > -999.0 ? exp2_f64_in(d) : 0.0;  // (NaN: 0)
    }
};

// The bin of n of a logit, 0 the highest: linear between `max` and `cut`.
// Rounded arithmetic, but monotonic: a higher logit is never in a lower bin.
// `inv` is 0, and all are in bin 0, where bins have no width in 32 bits or no
// reciprocal (logits closer than n / FLT_MAX).
struct Binner {
    float max, inv;
    int n;
    __device__ __forceinline__ Binner(float max_, float cut, int n_) : max(finite(max_)), n(n_)
    {
        const float width = max - cut;
        const float r = (float)n / width;
        inv = width > 0.0f && r < INFINITY ? r : 0.0f;
    }
    __device__ __forceinline__ int operator()(float l) const { return (int)fminf((max - finite(l)) * inv, (float)(n - 1)); }
};

// ------------------------------------------------- sums over the workgroup
// Lanes' values shifted within the wave, 0 where there is none: the steps of a
// running sum (within a row of 16 by 1, 2, 4, 8, then row 0's and 2's last
// lane to the next row, then lane 31 to the upper half).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v)
{
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_u64(double v)
{
    return __builtin_bit_cast(double, dpp_u64<CTRL, ROWS>(__builtin_bit_cast(uint64_t, v)));
}
template <class T>
__device__ __forceinline__ T wave_scan(T v)
{
    v += dpp_u64<0x111, 0xF>(v);
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    v += dpp_u64<0x142, 0xA>(v);
    v += dpp_u64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane)
{
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ double wave_sum_f64(double v)
{
    return __builtin_bit_cast(double, read_lane(__builtin_bit_cast(uint64_t, wave_scan(v)), 63));
}
// (least of the wave, in lane 63)
__device__ __forceinline__ uint64_t wave_min_u64(uint64_t v)
{
    v = ~v;  // (the shifts fill with 0, the least complement)
    auto up = [&](uint64_t o) { v = o > v ? o : v; };
    up(dpp_u64<0x111, 0xF>(v));
    up(dpp_u64<0x112, 0xF>(v));
    up(dpp_u64<0x114, 0xF>(v));
    up(dpp_u64<0x118, 0xF>(v));
    up(dpp_u64<0x142, 0xA>(v));
    up(dpp_u64<0x143, 0xC>(v));
    return ~v;
}

struct Scratch {
    uint64_t wave64[NW];
    uint64_t found[2];
    double wave_d[NW];
};

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
    v = wave_min_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wave64[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t m = sh.wave64[0];
#pragma unroll
    for (int i = 1; i < NW; i++) m = sh.wave64[i] < m ? sh.wave64[i] : m;
    return m;
}

// The thread at which the running sum of `mine` over the workgroup first
// reaches `limit` (>= 1), and the sum before it; -1 if it does not.
__device__ __forceinline__ int block_locate(Scratch& sh, uint64_t mine, uint64_t limit, uint64_t& before)
{
    uint64_t all;
    const uint64_t run = block_scan(sh, mine, all);
    if (all < limit) return -1;
    if (run >= limit && run - mine < limit) {
        sh.found[0] = threadIdx.x;
        sh.found[1] = run - mine;
    }
    __syncthreads();
    before = sh.found[1];
    return (int)(sh.found[0] & (NT - 1));
}

// What the units say of a row: its maximum and, of a sum over the whole row,
// Z; thread t holds units 2 t and 2 t + 1.
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
        if (2 * (threadIdx.x & ~63u) < (uint32_t)a.units)  // (not for waves without units)
#pragma unroll
            for (int i = 0; i < 2; i++) r.us[i] *= Weigher{r.max, s.c}(r.um[i]);  // (0: none of its entries weighs)
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
// The sum over a whole row is an exponential of 64 bits an entry, and those,
// not memory, bound this launch.  2^(j / 1024) comes from a table in LDS, which
// leaves f in [-1/2, 1/2] of a step: 2^(f / 1024) = 1 + f (K + f K^2 / 2), K =
// ln 2 / 1024, off by 7e-12 at its ends (odd in f, so that it averages out of a
// sum).  The table's upper words lack j << 10, so that n << 10 (n in steps, j its
// lower bits) makes index and exponent right at once.  7 operations of 64
// bits and a lookup, against 16 of exp2_f64.
constexpr int TABLE = 1024;
__device__ __forceinline__ double table_entry(int j)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, exp2_f64_in((double)j / TABLE));
    return __builtin_bit_cast(double, b - ((uint64_t)(uint32_t)j << 42));
}
// 2^(d * steps / 1024), |d * steps| < 2^20
__device__ __forceinline__ double exp2_table(const double* table, double d, double steps)
{
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    constexpr double K = 0.0006769015435155716;
    const double t = fma(d, steps, MAGIC);
    const double f = fma(d, steps, MAGIC - t);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    u32x2 e = __builtin_bit_cast(u32x2, table[n & (TABLE - 1)]);
    e.y += n << 10;
    const double r = __builtin_bit_cast(double, e);
    return fma(r, fma(f, K * K / 2, K) * f, r);
}

template <int LT>
__global__ void __launch_bounds__(NT, 8) sample_stats_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ double table[TABLE];
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    if (blockIdx.x == 0 && tid < CNTS) a.counters[b * CNTS + tid] = 0;
    const Row<LT> row(a, b);
    const int unit = blockIdx.x * NW + (tid >> 6);
    const int from = unit * a.unit_blocks + lane, end = min(row.blocks, (unit + 1) * a.unit_blocks);
    const u32x4 head = row.head(from, end);
    const Setting s(a, b);
    if (s.whole_sum()) {
        for (int i = tid; i < TABLE; i += NT) table[i] = table_entry(i);
        __syncthreads();
    }
    if (unit >= a.units) return;
    float m = -INFINITY;
    double sum = 0.0;
    if (s.whole_sum()) {
        // sum of exp((l - ref) / temperature), ref one of the lane's logits:
        // 64 bits hold weights of 2^1000, so it moves only where one is close,
        // past `high`, 900 binary orders above: a sum of weights up to there,
        // moved by the most that exp2_f64 takes away, 2^-1000, is nothing
        // beside a weight of 1.  Differences are held above -990 / c, whose weight is
        // nothing, by a median, which drops NaN as well as -inf: of 16-bit
        // logits in 32 bits, exact but for logits 2^-13 of ref and below; of
        // 32-bit ones before the difference in 64.  `quick` is whether fp32
        // has that bound (it does but for huge logits and temperatures).
        const double steps = s.c * TABLE;
        const float span = (float)fmin(900.0 / s.c, (double)FLT_MAX), lim = (float)fmin(990.0 / s.c, (double)FLT_MAX);
        float ref = -INFINITY, high = -INFINITY, least = -INFINITY;
        bool quick = false;
        row.stream(from, end, 64, head, [&](int, const float (&v)[VEC]) {
            float top = v[0];
#pragma unroll
            for (int j = 1; j < VEC; j++) top = fmaxf(top, v[j]);
            m = fmaxf(m, top);
            top = finite(top);
            if (top > high) {
                sum *= exp2_f64(((double)ref - (double)top) * s.c);
                ref = top;
                high = (float)fmin((double)ref + (double)span, (double)FLT_MAX);
                least = (float)fmax((double)ref - (double)lim, (double)-FLT_MAX);
                if (((double)high - (double)ref) * s.c > 910.0) high = ref;  // (rounded further up than that)
                quick = LT == VQ2_DT_F32 ? fabs(((double)ref - (double)least) * s.c - 990.0) < 5.0 : lim < 1e37f && ref < FLT_MAX;
            }
            if (quick) {
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    double d;
                    if constexpr (LT == VQ2_DT_F32)
                        d = (double)__builtin_amdgcn_fmed3f(v[j], least, FLT_MAX) - (double)ref;
                    else
                        d = (double)__builtin_amdgcn_fmed3f(v[j] - ref, -lim, lim);
                    sum += exp2_table(table, d, steps);
                }
            } else {
                for (int j = 0; j < VEC; j++) {
                    const double y = ((double)finite(v[j]) - (double)ref) * s.c;
                    sum += exp2_f64(y > 1000.0 ? 1000.0 : y);  // (NaN stays: 2^-1000)
                }
            }
        });
        const float um = wave_max_all(m);
        sum *= exp2_f64(((double)ref - (double)um) * s.c);
        if (um == INFINITY) {  // (the infinite ones count, and nothing else)
            sum = 0.0;
            row.stream(from, end, 64, [&](int, const float (&v)[VEC]) {
#pragma unroll
                for (int j = 0; j < VEC; j++) sum += v[j] == INFINITY ? 1.0 : 0.0;
            });
        }
        sum = wave_sum_f64(sum);
    } else {
        row.stream(from, end, 64, head, [&](int, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++) m = fmaxf(m, v[j]);
        });
    }
    const int64_t at = (int64_t)b * a.units + unit;
    if (s.k > 1) {
        float g = m;
        if (a.fine < 64) {
            g = fmaxf(g, dpp_xor1(g));
            g = fmaxf(g, dpp_xor2(g));
        }
        if (a.fine == 4) {
            g = fmaxf(g, dpp_half_mirror(g));
            g = fmaxf(g, dpp_row_mirror(g));
        }
        const int each = 64 / a.fine;
        if (lane % each == 0) a.fine_max[at * a.fine + lane / each] = g;
    }
    m = wave_max_all(m);
    if (lane == 0) {
        a.unit_max[at] = m;
        a.unit_sum[at] = sum;
    }
}

// ----------------------------------------------------------------- collect
// Entries of a workgroup on their way to a list.
struct Stage {
    uint64_t entry[LIST];
    uint32_t n, base;
};

// Puts the entries of this block that pass `in` into the stage (those past its
// end are counted only): the wave counts them by ballots and takes their places
// at once.
template <int VEC, class F>
__device__ __forceinline__ void stage_block(Stage& st, int block, const float (&v)[VEC], F in)
{
    uint64_t pass[VEC];
    uint32_t total = 0;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        pass[j] = __ballot(in(v[j]));
        total += (uint32_t)__popcll(pass[j]);
    }
    if (total == 0) return;
    const uint64_t active = __ballot(true);
    uint32_t at = 0;
    if (__builtin_amdgcn_mbcnt_hi((uint32_t)(active >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)active, 0)) == 0)
        at = atomicAdd(&st.n, total);
    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        if (pass[j] == 0) continue;
        const uint32_t to =
            at + __builtin_amdgcn_mbcnt_hi((uint32_t)(pass[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)pass[j], 0));
        if (in(v[j]) && to < LIST) st.entry[to] = order_key(v[j], block * VEC + j);
        at += (uint32_t)__popcll(pass[j]);
    }
}

// Appends the stage to a list of `cap` entries; the list's counter counts
// entries that do not fit as well.
__device__ __forceinline__ void flush_stage(Stage& st, uint32_t* counter, uint64_t* list, uint32_t cap)
{
    __syncthreads();
    const uint32_t n = st.n;
    if (n == 0) return;
    if (threadIdx.x == 0) st.base = atomicAdd(counter, n);
    __syncthreads();
    const uint32_t base = st.base;
    if (n > LIST || base > cap || n > cap - base) return;
    for (uint32_t i = threadIdx.x; i < n; i += NT) list[base + i] = st.entry[i];
}

// The smallest logit of weight >= min_p, by a search of 64 steps at once.
__device__ __forceinline__ float min_p_border(const Setting& s, const Weigher& weigh)
{
    uint32_t lo = 0x00800000u, hi = (uint32_t)(order_key(weigh.max, 0) >> 32);  // (-FLT_MAX's; weight 1 >= min_p)
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, probe = lo + min((threadIdx.x & 63) * step, hi - lo);
        const uint64_t yes = __ballot(weigh(key_logit((uint64_t)probe << 32)) >= s.min_p);
        if (yes == 0) {  // (the last probe is short of hi then)
            lo += 63 * step + 1;
        } else {
            const uint32_t f = (uint32_t)__ffsll((unsigned long long)yes) - 1, top = hi - lo;
            hi = lo + min(f * step, top);
            if (f > 0) lo += (f - 1) * step + 1;
        }
    }
    return key_logit((uint64_t)hi << 32);
}

struct CollectShared {
    Scratch scratch;
    Stage stage;
    uint64_t amount[BINS];
    uint32_t count[NT];
};

// The logit from which on a row's entries may stay: rounded down, by more than
// the arithmetic here is off.
__device__ float lowest_kept(CollectShared& sh, const SampleArgs& a, const Setting& s, const Units& un, int b)
{
    const int tid = threadIdx.x;
    if (un.max == INFINITY) return un.max;  // (no finite logit weighs anything)
    const double m = (double)un.max;
    // (the logarithm of 32 bits is off by less than 0.001)
    double bits = -45.0;
    if (s.k == 0 && s.top_p_on)
        bits = fmax(bits, (double)__builtin_amdgcn_logf((float)((1.0 - s.p) * un.z / (double)a.vocab)) - 0.002);
    double low = m + bits / s.c;
    low -= (fabs(m) + fabs(low)) * 1e-6;
    float cut = (float)fmax(low, (double)-FLT_MAX);
    if (s.k > 0) {
        // the lower end of the range that the k-th largest maximum falls into;
        // more groups than k are needed for it to say something
        const bool coarse = s.k * 2 <= (uint32_t)a.units;
        const int groups = coarse ? a.units : a.units * a.fine;
        if (s.k * 5 <= (uint32_t)groups * 4) {
            const int64_t u0 = (int64_t)b * a.units;
            const float* const from = coarse ? a.unit_max + u0 : a.fine_max + u0 * a.fine;
            float g[MAX_GROUPS / NT], least = INFINITY;  // (all loads in flight together)
#pragma unroll
            for (int i = 0; i < MAX_GROUPS / NT; i++) g[i] = tid + i * NT < groups ? from[tid + i * NT] : INFINITY;
#pragma unroll
            for (int i = 0; i < MAX_GROUPS / NT; i++) least = fminf(least, fmaxf(g[i], cut));
            least = -block_max(sh.scratch, -least);
            const Binner bin(un.max, least, NT);
            sh.count[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < MAX_GROUPS / NT; i++)
                if (tid + i * NT < groups && g[i] >= least) atomicAdd(&sh.count[bin(g[i])], 1u);
            __syncthreads();
            uint64_t before;
            const int r = block_locate(sh.scratch, sh.count[tid], s.k, before);
            // (the range's end as the binner rounds it, and a range to spare)
            if (r >= 0 && bin.inv > 0.0f) cut = fmaxf(cut, un.max - (float)(r + 2) / bin.inv);
        }
    }
    if (s.min_p_on && !(s.k > 0 && s.top_p_on)) {
        __syncthreads();
        if (tid < 64) {
            const float at = min_p_border(s, Weigher{un.max, s.c});
            if (tid == 0) sh.scratch.wave_d[0] = (double)at;
        }
        __syncthreads();
        cut = fmaxf(cut, (float)sh.scratch.wave_d[0]);
    }
    return cut;
}

template <int LT>
__global__ void __launch_bounds__(NT, 8) sample_collect_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ CollectShared sh;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const Setting s(a, b);
    if (!s.listed()) return;
    const Units un = read_units(sh.scratch, a, s, b);
    if (un.max == -INFINITY) return;
    const float cut = lowest_kept(sh, a, s, un, b);
    if (blockIdx.x == 0 && tid == 0) a.info[b] = RowInfo{un.z, un.max, cut};
    const Row<LT> row(a, b);
    const int unit = blockIdx.x * NW + (tid >> 6);
    const int from = unit * a.unit_blocks, end = min(row.blocks, from + a.unit_blocks);
    if (tid == 0) sh.stage.n = 0;
    __syncthreads();
    row.stream(from + lane, end, 64, [&](int i, const float (&v)[VEC]) {
        float top = v[0];
#pragma unroll
        for (int j = 1; j < VEC; j++) top = fmaxf(top, v[j]);
        if (__ballot(top >= cut)) stage_block<VEC>(sh.stage, i, v, [&](float l) { return l >= cut; });
    });
    __syncthreads();
    const uint32_t n = sh.stage.n;
    const bool is_long = n > a.short_slice();
    const int64_t slice = (int64_t)b * gridDim.x + blockIdx.x;
    if (tid == 0) a.slice_n[slice] = n;
    if (is_long)
        flush_stage(sh.stage, a.counters + b * CNTS + CNT_LONG, a.list + (int64_t)b * a.list_cap, a.list_cap);
    else
        flush_stage(sh.stage, a.counters + b * CNTS + CNT_SHORT, a.short_list + (int64_t)b * a.short_cap, a.short_cap);
    if (!is_long) return;
    // a histogram of the slice's entries, in case the row has too many
    if (tid < BINS) {
        sh.amount[tid] = 0;
        sh.count[tid] = 0;
    }
    __syncthreads();
    const Weigher weigh{un.max, s.c};
    const Binner bin(un.max, cut, BINS);
    auto add = [&](float l) {
        const int r = bin(l);
        atomicAdd((unsigned long long*)&sh.amount[r], (unsigned long long)fixed(weigh(l)));
        atomicAdd(&sh.count[r], 1u);
    };
    if (n <= LIST) {
        for (uint32_t i = tid; i < n; i += NT) add(key_logit(sh.stage.entry[i]));
    } else {
        row.stream(from + lane, end, 64, [&](int, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (v[j] >= cut) add(v[j]);
        });
    }
    __syncthreads();
    if (tid < BINS) {
        a.bin_amount[slice * BINS + tid] = sh.amount[tid];
        a.bin_count[slice * BINS + tid] = sh.count[tid];
    }
}

// ------------------------------------------------------------------ refine
struct RefineShared {
    Scratch scratch;
    uint32_t is_long[MAX_UNITS / NW];
    Stage stage;
    uint64_t amount[NT];
    uint32_t count[NT];
};

template <int LT>
__global__ void __launch_bounds__(NT, 8) sample_refine_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ RefineShared sh;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, slices = a.slices();
    const uint32_t n_long = a.counters[b * CNTS + CNT_LONG], n_short = a.counters[b * CNTS + CNT_SHORT];
    if (n_long + n_short <= LIST) return;
    const Setting s(a, b);
    if (!s.one_border()) return;
    const RowInfo info = a.info[b];
    const Weigher weigh{info.max, s.c};
    const Binner bin(info.max, info.cut, BINS);
    // the row's histogram: two bins a thread of every fourth slice, eight
    // slices' loads in flight, then the short slices' entries
    const int64_t slice0 = (int64_t)b * slices;
    sh.amount[tid] = 0;
    sh.count[tid] = 0;
    if (tid < slices) sh.is_long[tid] = a.slice_n[slice0 + tid] > a.short_slice();
    __syncthreads();
    {
        constexpr int PAIRS = BINS / 2;
        const int pair = tid % PAIRS;
        uint64_t am[2] = {};
        uint32_t ct[2] = {};
#pragma unroll 8
        for (int g = tid / PAIRS; g < slices; g += NT / PAIRS) {
            // (a short slice's, which nothing wrote, are loaded and dropped: no branch keeps the loads apart)
            const ulonglong2 x = ((const ulonglong2*)a.bin_amount)[(slice0 + g) * PAIRS + pair];
            const uint2 y = ((const uint2*)a.bin_count)[(slice0 + g) * PAIRS + pair];
            const bool is_long = sh.is_long[g] != 0;
            am[0] += is_long ? x.x : 0;
            am[1] += is_long ? x.y : 0;
            ct[0] += is_long ? y.x : 0;
            ct[1] += is_long ? y.y : 0;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            atomicAdd((unsigned long long*)&sh.amount[2 * pair + i], (unsigned long long)am[i]);
            atomicAdd(&sh.count[2 * pair + i], ct[i]);
        }
        for (uint32_t i = tid; i < min(n_short, (uint32_t)a.short_cap); i += NT) {
            const float l = key_logit(a.short_list[(int64_t)b * a.short_cap + i]);
            atomicAdd((unsigned long long*)&sh.amount[bin(l)], (unsigned long long)fixed(weigh(l)));
            atomicAdd(&sh.count[bin(l)], 1u);
        }
    }
    __syncthreads();
    const double p_limit = ceil(s.p * info.z * UNIT);
    const uint64_t limit = s.k > 0 ? (uint64_t)s.k : !s.top_p_on ? ~0ull : p_limit > 1.0 ? (uint64_t)p_limit : 1;
    const uint64_t amount = tid < BINS ? (s.k > 0 ? (uint64_t)sh.count[tid] : sh.amount[tid]) : 0;
    uint64_t before = 0;
    const int r = block_locate(sh.scratch, amount, limit, before);
    if (blockIdx.x == 0 && tid == 0) a.refined[b] = RefineInfo{before, r};
    const Row<LT> row(a, b);
    for (int g = blockIdx.x; g < slices; g += gridDim.x) {
        if (a.slice_n[slice0 + g] <= a.short_slice()) continue;
        // the slice's weight ahead of the bin, and its entries of the bin
        const uint64_t ahead = tid < BINS && (r < 0 || tid < r) ? a.bin_amount[(slice0 + g) * BINS + tid] : 0;
        uint64_t all;
        block_scan(sh.scratch, ahead, all);
        if (tid == 0) a.slice_mass[slice0 + g] = all;
        if (r < 0) continue;
        if (tid == 0) sh.stage.n = 0;
        __syncthreads();
        const int from = (g * NW + (tid >> 6)) * a.unit_blocks, end = min(row.blocks, from + a.unit_blocks);
        row.stream(from + lane, end, 64, [&](int i, const float (&v)[VEC]) {
            stage_block<VEC>(sh.stage, i, v, [&](float l) { return l >= info.cut && bin(l) == r; });
        });
        flush_stage(sh.stage, a.counters + b * CNTS + CNT_BIN, a.list + (int64_t)b * a.list_cap, a.list_cap);
    }
}

// ------------------------------------------------------------------ finish
struct FinishShared {
    Scratch scratch;
    uint64_t list[LIST];  // entries
    uint64_t mass[LIST];  // and their weights
    uint64_t amount[NT];  // a histogram's sums, or entries that are ranked: amounts,
    uint64_t order[NT];   // places
    uint32_t index[NT];   // and which they are
    uint32_t count[NT];   // a histogram's entries
    uint64_t slice[MAX_UNITS / NW];
    uint32_t n;
};

// Of entries 0 ... n - 1 with different places order(i) (ascending), the one
// at which the running sum of amount(i), in their order, first reaches `limit`
// (>= 1); -1 if it does not.  A histogram over ranges of the order, bin(i) <
// NT, finds the range; while that holds more than DIRECT entries, it is cut
// into NT equal ranges again (places differ, so that ends).  The entries left
// are compared with each other.
template <class Order, class Amount, class Bin>
__device__ __forceinline__ int locate_entry(FinishShared& sh, int n, uint64_t limit, Order order, Amount amount, Bin bin)
{
    const int tid = threadIdx.x;
    uint64_t lo = 0, hi = ~0ull, before = 0;
    int shift = -1;  // (the first round: bin)
    for (;;) {
        auto range = [&](int i) -> int {
            if (shift < 0) return bin(i);
            const uint64_t o = order(i);
            return o < lo || o > hi ? -1 : (int)((o - lo) >> shift);
        };
        __syncthreads();
        sh.amount[tid] = 0;
        sh.count[tid] = 0;
        if (tid == 0) sh.n = 0;
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
            const uint64_t x = amount(i);
            const int r = range(i);
            if (x && r >= 0) {
                atomicAdd((unsigned long long*)&sh.amount[r], (unsigned long long)x);
                atomicAdd(&sh.count[r], 1u);
            }
        }
        __syncthreads();
        uint64_t ahead = 0;
        const int at = block_locate(sh.scratch, sh.amount[tid], limit - before, ahead);
        if (at < 0) return -1;
        before += ahead;
        const uint32_t m = sh.count[at];
        __syncthreads();
        if (m <= DIRECT || shift == 0) {
            // gather, then compare
            for (int i = tid; i < n; i += NT) {
                const uint64_t x = amount(i);
                if (x && range(i) == at) {
                    const uint32_t to = atomicAdd(&sh.n, 1u) & (NT - 1);
                    sh.amount[to] = x;
                    sh.order[to] = order(i);
                    sh.index[to] = (uint32_t)i;
                }
            }
            __syncthreads();
            if (tid < (int)min(m, (uint32_t)NT)) {
                const uint64_t o = sh.order[tid];
                uint64_t ahead_of = before;
#pragma unroll 8
                for (uint32_t j = 0; j < m; j++) ahead_of += sh.order[j] < o ? sh.amount[j] : 0;
                if (ahead_of < limit && ahead_of + sh.amount[tid] >= limit) sh.scratch.found[0] = sh.index[tid];
            }
            __syncthreads();
            return (int)sh.scratch.found[0];
        }
        // the places that the range spans
        uint64_t least = ~0ull, most = ~0ull;
        for (int i = tid; i < n; i += NT)
            if (amount(i) && range(i) == at) {
                const uint64_t o = order(i);
                least = o < least ? o : least;
                most = ~o < most ? ~o : most;
            }
        least = block_min(sh.scratch, least);
        most = ~block_min(sh.scratch, most);
        lo = least;
        hi = most;
        shift = hi - lo < NT ? 0 : 64 - __clzll(hi - lo) - BITS;
    }
}

__device__ __forceinline__ double clamped_u(const SampleArgs& a, int b) { return fmin(fmax((double)a.u[b], 0.0), 1.0); }

// u of the total, plus one: the running sum that the token's reaches first.
__device__ __forceinline__ uint64_t draw_limit(const SampleArgs& a, int b, uint64_t total)
{
    const uint64_t t = (uint64_t)(clamped_u(a, b) * (double)total);
    return t < total ? t + 1 : total;
}

__device__ __forceinline__ void write_token(const SampleArgs& a, int b, int column, float l, const Weigher& weigh,
                                            double total)
{
    a.out_idx[b] = column;
    a.out_logprob[b] = (float)(weigh.log2_of(l) / LOG2E_F64 - log(total));
}

// Up to DIRECT entries: each one's rank and the weight ahead of it, and the
// kept weight of lower columns, by comparing it with every other, a part of
// them by each of its threads.  (The comparisons are what it costs: over 250
// entries they took 5 us, and finish_list's histograms 4, hence DIRECT.)
__device__ __forceinline__ void finish_direct(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh,
                                              int n, double z, int b)
{
    const int tid = threadIdx.x, i = tid & (DIRECT - 1), part = tid / DIRECT;
    const int j0 = part * n / PARTS, j1 = (part + 1) * n / PARTS;
    const uint64_t key = i < n ? sh.list[i] : 0, mass = i < n ? sh.mass[i] : 0;
    uint32_t rank = 0;
    uint64_t before = 0;
    if (i - (tid & 63) < n)  // (waves without an entry)
#pragma unroll 8
        for (int j = j0; j < j1; j++) {
            const bool ahead = sh.list[j] > key;
            rank += ahead;
            before += ahead ? sh.mass[j] : 0;
        }
    sh.order[tid] = before;
    sh.count[tid] = rank;
    __syncthreads();
    rank = 0;
    before = 0;
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
        rank += sh.count[p * DIRECT + i];
        before += sh.order[p * DIRECT + i];
    }
    bool stays = i < n && (s.k == 0 || rank < s.k);
    uint64_t total;
    if (s.top_p_on) {
        double all = z * UNIT;
        if (s.k > 0) {
            block_scan(sh.scratch, part == 0 && stays ? mass : 0, total);
            all = (double)total;
        }
        stays = stays && (rank == 0 || (double)before < s.p * all);
    }
    if (s.min_p_on) stays = stays && weigh(key_logit(key)) >= s.min_p;
    const uint64_t kept = stays ? mass : 0;
    if (part == 0) sh.amount[i] = kept;
    block_scan(sh.scratch, part == 0 ? kept : 0, total);  // (its barriers are amount's and order's as well)
    const uint64_t limit = draw_limit(a, b, total);
    uint64_t run = 0;
    const uint32_t col = ~(uint32_t)key;
    if (i - (tid & 63) < n)
#pragma unroll 8
        for (int j = j0; j < j1; j++) run += ~(uint32_t)sh.list[j] < col ? sh.amount[j] : 0;
    sh.order[tid] = run;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int p = 1; p < PARTS; p++) run += sh.order[p * DIRECT + i];
    if (kept && run < limit && run + kept >= limit)
        write_token(a, b, key_column(key), key_logit(key), weigh, (double)total / UNIT);
}

// A list of more entries: the borders by the order of logits, the draw by the
// order of columns.
__device__ __forceinline__ void finish_list(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh, int n,
                                            float cut, double z, int b)
{
    const Binner bin(weigh.max, cut, NT);
    uint64_t lo = 0, total;
    for (int by_mass = s.k == 0; by_mass <= (int)s.top_p_on; by_mass++) {  // top-k, top-p
        double limit = (double)s.k;
        if (by_mass) {
            limit = z * UNIT;
            if (s.k > 0) {
                uint64_t part = 0;
                for (int i = threadIdx.x; i < n; i += NT) part += sh.list[i] >= lo ? sh.mass[i] : 0;
                block_scan(sh.scratch, part, total);
                limit = (double)total;
            }
            limit = fmax(1.0, ceil(s.p * limit));
        }
        const int at = locate_entry(
            sh, n, (uint64_t)limit, [&](int i) { return ~sh.list[i]; },
            [&](int i) -> uint64_t { return sh.list[i] < lo ? 0 : by_mass ? sh.mass[i] : 1; },
            [&](int i) { return bin(key_logit(sh.list[i])); });
        if (at >= 0) lo = sh.list[at];
    }
    // what does not stay weighs nothing from here on
    uint64_t part = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t key = sh.list[i];
        if (key < lo || (s.min_p_on && !(weigh(key_logit(key)) >= s.min_p))) sh.mass[i] = 0;
        part += sh.mass[i];
    }
    block_scan(sh.scratch, part, total);
    const int width = (a.vocab + NT - 1) / NT;
    const int at = locate_entry(
        sh, n, draw_limit(a, b, total), [&](int i) { return (uint64_t)(uint32_t)~(uint32_t)sh.list[i]; },
        [&](int i) { return sh.mass[i]; }, [&](int i) { return key_column(sh.list[i]) / width; });
    if (threadIdx.x == 0)
        write_token(a, b, key_column(sh.list[at]), key_logit(sh.list[at]), weigh, (double)total / UNIT);
}

// A row after the refine launch: the border among its bin's entries, then the
// slice that the draw falls into, whose entries are read again.  False if the
// bin has too many.
template <int LT>
__device__ __forceinline__ bool finish_refined(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh,
                               const Row<LT>& row, const RowInfo& info, uint32_t n_short, int b)
{
    constexpr int VEC = Row<LT>::VEC;
    const int tid = threadIdx.x, slices = a.slices();
    const int64_t slice0 = (int64_t)b * slices;
    const RefineInfo ref = a.refined[b];
    const uint32_t n_bin = a.counters[b * CNTS + CNT_BIN];
    if (ref.bin >= 0 && n_bin > LIST) return false;
    const Binner bins(weigh.max, info.cut, BINS);
    const uint64_t* const short_list = a.short_list + (int64_t)b * a.short_cap;
    auto mass = [&](uint64_t key) { return fixed(weigh(key_logit(key))); };
    uint64_t lo = 0;
    int n = 0;
    if (ref.bin >= 0) {
        n = (int)n_bin;
        for (int i = tid; i < n; i += NT) sh.list[i] = a.list[(int64_t)b * a.list_cap + i];
        if (tid == 0) sh.n = n_bin;
        __syncthreads();
        for (uint32_t i = tid; i < n_short; i += NT) {
            const uint64_t key = short_list[i];
            if (bins(key_logit(key)) == (int)ref.bin) {
                const uint32_t to = atomicAdd(&sh.n, 1u);
                if (to < LIST) sh.list[to] = key;
            }
        }
        __syncthreads();
        if (sh.n > LIST) return false;
        n = (int)sh.n;
        for (int i = tid; i < n; i += NT) sh.mass[i] = mass(sh.list[i]);
        __syncthreads();
        // the bin's own range in NT
        const float top = weigh.max - (float)ref.bin / bins.inv, step = 1.0f / bins.inv;
        const Binner bin(top, top - step, NT);
        const double p_limit = ceil(s.p * info.z * UNIT);
        const uint64_t limit = s.k > 0 ? (uint64_t)s.k : p_limit > 1.0 ? (uint64_t)p_limit : 1;
        const int at = locate_entry(
            sh, n, limit - ref.before, [&](int i) { return ~sh.list[i]; },
            [&](int i) -> uint64_t { return s.k > 0 ? 1 : sh.mass[i]; },
            [&](int i) { return max(0, bin(key_logit(sh.list[i]))); });
        if (at >= 0) lo = sh.list[at];
    }
    // each slice's kept weight
    const int slice_cols = NW * a.unit_blocks * VEC;
    __syncthreads();
    if (tid < slices) {
        const uint32_t sn = a.slice_n[slice0 + tid];
        sh.slice[tid] = sn > a.short_slice() ? a.slice_mass[slice0 + tid] : 0;
        sh.count[tid] = sn > a.short_slice();
    }
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
        const uint64_t key = sh.list[i];
        const int g = key_column(key) / slice_cols;
        if (key >= lo && sh.count[g]) atomicAdd((unsigned long long*)&sh.slice[g], (unsigned long long)sh.mass[i]);
    }
    for (uint32_t i = tid; i < n_short; i += NT) {
        const uint64_t key = short_list[i];
        if (key >= lo) atomicAdd((unsigned long long*)&sh.slice[key_column(key) / slice_cols], (unsigned long long)mass(key));
    }
    __syncthreads();
    uint64_t total, before = 0, all;
    const uint64_t mine = tid < slices ? sh.slice[tid] : 0;
    block_scan(sh.scratch, mine, total);
    const uint64_t limit = draw_limit(a, b, total);
    const int g = block_locate(sh.scratch, mine, limit, before);
    // that slice, in pieces of the threads
    const int b0 = g * NW * a.unit_blocks, per = (NW * a.unit_blocks + NT - 1) / NT;
    const int i0 = b0 + tid * per, i1 = min(min(row.blocks, b0 + NW * a.unit_blocks), i0 + per);
    auto kept = [&](float l, int c) -> uint64_t { return l >= info.cut && order_key(l, c) >= lo ? fixed(weigh(l)) : 0; };
    uint64_t part = 0;
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++) part += kept(v[j], i * VEC + j);
    });
    uint64_t run = before + block_scan(sh.scratch, part, all);
    if (!(run >= limit && run - part < limit)) return true;
    run -= part;
    int col = 0;
    float l = weigh.max;
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (run < limit) {
                run += kept(v[j], i * VEC + j);
                col = i * VEC + j;
                l = v[j];
            }
    });
    write_token(a, b, col, l, weigh, (double)total / UNIT);
    return true;
}

// The last key that stays of a row of which nothing shorter is known (long ties
// in the border's bin; a long row under both top-k and top-p): a histogram
// finds a range of the order, and once a range's entries fit the list they are
// taken from it.  Passes over the row are what it costs: two for a range that
// fits at once, two more for one that holds too many (to find what it spans,
// and to cut that).  `known` is a bin of BINS that the border is already known
// to lie in, and the amount ahead of it.
template <int LT>
__device__ __forceinline__ uint64_t row_border(FinishShared& sh, const Row<LT>& row, float cut, const Weigher& weigh,
                                               uint64_t limit, bool by_mass, uint64_t from, const RefineInfo& known)
{
    constexpr int VEC = Row<LT>::VEC;
    const int tid = threadIdx.x;
    const Binner bin(weigh.max, cut, known.bin >= 0 ? BINS : NT);
    uint64_t lo = from, hi = ~0ull, before = known.bin >= 0 ? known.before : 0;
    int shift = -1, at = (int)known.bin;  // (the first round: bin)
    auto mass = [&](float l) -> uint64_t { return by_mass ? fixed(weigh(l)) : 1; };
    // f(range, key, logit) for the entries of the ranges (one compute unit's
    // arithmetic is what a pass costs: keys only of logits in between)
    auto entries = [&](auto f) {
        const float least = fmaxf(cut, lo ? key_logit(lo) : -INFINITY), most = hi == ~0ull ? INFINITY : key_logit(hi);
        row.stream_wide(tid, row.blocks, NT, [&](int i, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                if (!(v[j] >= least && v[j] <= most)) continue;
                const uint64_t key = order_key(v[j], i * VEC + j);
                if (key >= lo && key <= hi) f(shift < 0 ? bin(v[j]) : (int)((hi - key) >> shift), key, v[j]);
            }
        });
    };
    for (bool find = at < 0;; find = true) {
        if (find) {
            __syncthreads();
            sh.amount[tid] = 0;
            sh.count[tid] = 0;
            if (tid == 0) sh.n = 0;
            __syncthreads();
            // (runs of one range are added at once: ties would queue for it)
            int run = -1;
            uint64_t sum = 0;
            uint32_t length = 0;
            auto add = [&]() {
                atomicAdd((unsigned long long*)&sh.amount[run], (unsigned long long)sum);
                atomicAdd(&sh.count[run], length);
            };
            entries([&](int r, uint64_t, float l) {
                if (r != run) {
                    if (run >= 0) add();
                    run = r;
                    sum = 0;
                    length = 0;
                }
                sum += mass(l);
                length++;
            });
            if (run >= 0) add();
            __syncthreads();
            uint64_t ahead = 0;
            at = block_locate(sh.scratch, sh.amount[tid], limit - before, ahead);
            if (at < 0) return from;
            before += ahead;
            if (sh.count[at] <= LIST) break;
        }
        uint64_t least = ~0ull, most = ~0ull;  // (most: the largest key's complement)
        entries([&](int r, uint64_t key, float) {
            if (r != at) return;
            least = key < least ? key : least;
            most = ~key < most ? ~key : most;
        });
        lo = block_min(sh.scratch, least);
        hi = ~block_min(sh.scratch, most);
        if (lo > hi) return from;
        shift = hi - lo < NT ? 0 : 64 - __clzll(hi - lo) - BITS;
    }
    entries([&](int r, uint64_t key, float l) {
        if (r != at) return;
        const uint32_t to = atomicAdd(&sh.n, 1u);
        if (to >= LIST) return;
        sh.list[to] = key;
        sh.mass[to] = mass(l);
    });
    __syncthreads();
    const int n = (int)min(sh.n, (uint32_t)LIST);
    const int i = locate_entry(
        sh, n, limit - before, [&](int e) { return ~sh.list[e]; }, [&](int e) { return sh.mass[e]; }, [](int) { return 0; });
    return i >= 0 ? sh.list[i] : from;
}

template <int LT>
__device__ __forceinline__ void finish_row(FinishShared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh, const Row<LT>& row,
                           float cut, double z, const RefineInfo& known, int b)
{
    constexpr int VEC = Row<LT>::VEC;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    uint64_t lo = 0, total = 0;
    float least = cut;  // (and lo's logit: keys only of its ties)
    auto kept = [&](float l, int c, bool with_min) -> uint64_t {
        if (!(l >= least) || (l == least && order_key(l, c) < lo)) return 0;
        const double w = weigh(l);
        return with_min && s.min_p_on && !(w >= s.min_p) ? 0 : fixed(w);
    };
    // the kept weight of the wave's eighth of the row, which `range` cuts out
    const int eighth = (row.blocks + NW - 1) / NW;
    auto sum = [&](bool with_min) {
        uint64_t part = 0;
        row.stream_wide(wave * eighth + lane, min(row.blocks, (wave + 1) * eighth), 64, [&](int i, const float (&v)[VEC]) {
#pragma unroll
            for (int j = 0; j < VEC; j++) part += kept(v[j], i * VEC + j, with_min);
        });
        return part;
    };
    uint64_t part = 0;
    // top-k's border; the weight that it keeps, top-p's border; the kept weight
    for (int step = s.k > 0 ? 0 : s.top_p_on ? 2 : 3; step < 4; step++) {
        if (step == 1 || step == 3) {
            part = sum(step == 3);
            block_scan(sh.scratch, part, total);
            if (step == 1 && !s.top_p_on) step = 2;
            continue;
        }
        const double limit = step == 0 ? (double)s.k : fmax(1.0, ceil(s.p * (s.k > 0 ? (double)total : z * UNIT)));
        lo = row_border(sh, row, cut, weigh, (uint64_t)limit, step == 2, lo, known);
        if (lo) least = fmaxf(cut, key_logit(lo));
    }
    const uint64_t limit = draw_limit(a, b, total);
    uint64_t before = 0, all;
    const int w = block_locate(sh.scratch, part, limit, before) >> 6;
    // (the sum before the wave, not before its lane: the columns alternate between lanes)
    const uint64_t wave_sum = read_lane(wave_scan(part), 63);
    __syncthreads();
    if (lane == 63) sh.scratch.wave64[wave] = wave_sum;
    __syncthreads();
    before = 0;
    for (int i = 0; i < w; i++) before += sh.scratch.wave64[i];
    const int per = (eighth + NT - 1) / NT, i0 = w * eighth + tid * per;
    const int i1 = min(min(row.blocks, (w + 1) * eighth), i0 + per);
    uint64_t mine = 0;
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++) mine += kept(v[j], i * VEC + j, true);
    });
    uint64_t run = before + block_scan(sh.scratch, mine, all);
    if (!(run >= limit && run - mine < limit)) return;
    run -= mine;
    int col = 0;
    float l = weigh.max;
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (run < limit) {
                run += kept(v[j], i * VEC + j, true);
                col = i * VEC + j;
                l = v[j];
            }
    });
    write_token(a, b, col, l, weigh, (double)total / UNIT);
}

// A draw over the whole row: the unit, then the column, whose running sum is
// the first above u Z (the last with a weight, if rounding leaves none).
template <int LT>
__device__ __forceinline__ void finish_plain(FinishShared& sh, const SampleArgs& a, const Weigher& weigh, const Row<LT>& row, const Units& un,
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
        sh.scratch.found[0] = (uint64_t)(2 * t + second);
        sh.scratch.found[1] = __builtin_bit_cast(uint64_t, second ? before + un.us[0] : before);
    }
    __syncthreads();
    const int unit = (int)sh.scratch.found[0];
    const double base = __builtin_bit_cast(double, sh.scratch.found[1]);
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
    row.stream(i0, i1, 1, [&](int i, const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            if (col >= 0 && before > target) continue;
            const double w = weigh(v[j]);
            before += w;
            if (w > 0.0) {
                col = i * VEC + j;
                l = v[j];
            }
        }
    });
    write_token(a, b, col, l, weigh, un.z);
}

template <int LT>
__global__ void __launch_bounds__(NT, 4) sample_finish_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ FinishShared sh;
    const int b = blockIdx.x, tid = threadIdx.x;
    const Setting s(a, b);
    const Row<LT> row(a, b);
    if (!s.listed()) {
        const Units un = read_units(sh.scratch, a, s, b);
        const Weigher weigh{un.max, s.c};
        if (un.max == -INFINITY) {
            if (tid == 0) {
                a.out_idx[b] = -1;
                a.out_logprob[b] = NAN;
            }
        } else if (s.k == 1) {  // the first maximum
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
        } else {
            finish_plain<LT>(sh, a, weigh, row, un, b);
        }
        return;
    }
    const uint32_t n_long = a.counters[b * CNTS + CNT_LONG], n_short = a.counters[b * CNTS + CNT_SHORT];
    const uint32_t n = n_long + n_short;
    if (n == 0) {  // (nothing collected: the row has no maximum)
        if (tid == 0) {
            a.out_idx[b] = -1;
            a.out_logprob[b] = NAN;
        }
        return;
    }
    const RowInfo info = a.info[b];
    const Weigher weigh{info.max, s.c};
    if (n <= LIST) {
        for (uint32_t i = tid; i < n; i += NT) {
            const uint64_t key = i < n_long ? a.list[(int64_t)b * a.list_cap + i]
                                            : a.short_list[(int64_t)b * a.short_cap + (i - n_long)];
            sh.list[i] = key;
            sh.mass[i] = fixed(weigh(key_logit(key)));
        }
        __syncthreads();
        if (n <= DIRECT)
            finish_direct(sh, a, s, weigh, (int)n, info.z, b);
        else
            finish_list(sh, a, s, weigh, (int)n, info.cut, info.z, b);
        return;
    }
    const bool refined = a.refines && s.one_border();
    if (refined && finish_refined<LT>(sh, a, s, weigh, row, info, n_short, b)) return;
    __syncthreads();
    finish_row<LT>(sh, a, s, weigh, row, info.cut, info.z, refined ? a.refined[b] : RefineInfo{0, -1}, b);
}

// How a call is cut: units of at least 64 blocks (one load a lane), longer
// ones where the rows alone fill the device, 8192 waves of up to 64 registers.
struct Plan {
    int units, unit_blocks, fine, list_cap, short_cap;
    size_t unit_sum, unit_max, fine_max, counters, info, refined, slice_n, slice_mass, bin_amount, bin_count, list,
        short_list, bytes;
};

Plan make_plan(int64_t rows, int64_t vocab, int vec)
{
    Plan p;
    const int64_t blocks = (vocab + vec - 1) / vec;
    int64_t per = (blocks * rows + 8191) / 8192;
    per = per > (blocks + MAX_UNITS - 1) / MAX_UNITS ? per : (blocks + MAX_UNITS - 1) / MAX_UNITS;
    per = per > (blocks + NW - 1) / NW ? (blocks + NW - 1) / NW : per;
    p.unit_blocks = (int)((per + 63) / 64 * 64);
    p.units = (int)((blocks + p.unit_blocks - 1) / p.unit_blocks);
    p.fine = p.units < 128 ? 64 : p.units < 512 ? 16 : 4;
    p.list_cap = vocab < LIST ? (int)vocab : LIST;
    p.short_cap = vocab < SHORT_LIST ? (int)vocab : SHORT_LIST;
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
    p.counters = take(rows * CNTS * 4);
    p.info = take(rows * sizeof(RowInfo));
    p.refined = take(rows * sizeof(RefineInfo));
    p.slice_n = take(slices * 4);
    p.slice_mass = take(slices * 8);
    p.bin_amount = take(slices * BINS * 8);
    p.bin_count = take(slices * BINS * 4);
    p.list = take(rows * p.list_cap * 8);
    p.short_list = take(rows * p.short_cap * 8);
    p.bytes = at;
    return p;
}

template <int LT>
int launch(const SampleCall& c)
{
    const Plan p = make_plan(c.rows, c.vocab, Row<LT>::VEC);
    char* const ws = (char*)c.workspace;
    // settings common to all rows say here which launches have nothing to do:
    // without a border nothing is listed; no list is long where the row is
    // short or a top-k of at most LIST / 3 cuts it (but for ties, which the
    // finish goes over by itself)
    const bool by_row = c.temperature_rows || c.top_k_rows || c.top_p_rows || c.min_p_rows;
    const bool listed = by_row || (c.temperature > 0.0f && c.top_k != 1 && (c.top_k > 0 || c.top_p < 1.0f || c.min_p > 0.0f));
    const bool refine = listed && c.vocab > LIST && (by_row || c.top_k == 0 || c.top_k > LIST / 3);
    const SampleArgs a{c.logits, c.l_stride, (int)c.vocab, p.units, p.unit_blocks, p.fine, p.list_cap, p.short_cap, refine,
                       c.u, c.temperature_rows, c.top_k_rows, c.top_p_rows, c.min_p_rows,
                       c.temperature, c.top_p, c.min_p, c.top_k, c.out_idx, c.out_logprob,
                       (double*)(ws + p.unit_sum), (float*)(ws + p.unit_max), (float*)(ws + p.fine_max),
                       (uint32_t*)(ws + p.counters), (RowInfo*)(ws + p.info), (RefineInfo*)(ws + p.refined),
                       (uint32_t*)(ws + p.slice_n), (uint64_t*)(ws + p.slice_mass), (uint64_t*)(ws + p.bin_amount),
                       (uint32_t*)(ws + p.bin_count), (uint64_t*)(ws + p.list), (uint64_t*)(ws + p.short_list)};
    hipStream_t st = (hipStream_t)c.stream;
    const dim3 grid((unsigned)((p.units + NW - 1) / NW), (unsigned)c.rows), block(NT);
    hipLaunchKernelGGL(sample_stats_kernel<LT>, grid, block, 0, st, a);
    if (listed) hipLaunchKernelGGL(sample_collect_kernel<LT>, grid, block, 0, st, a);
    if (refine) {  // (rows mostly leave at once: no more workgroups than spread a single long row)
        const unsigned per_row = (unsigned)(c.rows < 512 ? 512 / c.rows : 1);
        hipLaunchKernelGGL(sample_refine_kernel<LT>, dim3(per_row < grid.x ? per_row : grid.x, grid.y), block, 0, st, a);
    }
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
