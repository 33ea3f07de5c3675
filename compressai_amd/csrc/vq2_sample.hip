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
// Two launches.  A row is cut into units, each a contiguous piece that one
// wave reads; the first launch leaves every unit's maximum and weight (and,
// for top-k, the maxima of finer groups).  The second knows the row's maximum
// and total from them and with them a logit below which nothing can stay:
//   top-k    the k-th largest of the groups' maxima (k entries are that large)
//   top-p    w < (1 - p) Z / V: all such entries together weigh less than
//            (1 - p) Z, which the last entries may be short of
//   min-p    w < min_p;  always: w < 2^-45
// It writes the entries above (usually some hundred to some thousand of the
// row) to a list, in column order, and the row's last workgroup finishes on it
// in LDS: a histogram of the order's keys narrows the border down to 128
// entries, which are ranked directly, then a running sum over the list finds
// the token.  A row whose list is too long (flat rows, long ties) is finished
// from the logits themselves by the same code.  A draw without a border (no
// top-k or top-p or min-p) needs one unit read again, whose weights' sum
// passes u Z.
#include <float.h>

#include "vq2_common.hpp"
#include "vq2_router.hpp"
#include "vq2_internal.hpp"

namespace vq2 {

namespace {

constexpr int NT = 1024;          // threads of a workgroup
constexpr int NW = NT / 64;       // its waves, one unit each
constexpr int MAX_UNITS = 1024;   // units of a row
constexpr int LIST = 6144;        // entries of the list in LDS
constexpr int DIRECT = 128;       // entries that are ranked directly
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
    uint32_t* arrivals;   // [rows]
    double* unit_sum;     // [rows][units], of exp((l - unit's max) / temperature)
    float* unit_max;      // [rows][units]
    float* fine_max;      // [rows][units][fine]
    uint32_t* list_len;   // [rows][units]
    uint64_t* list;       // [rows][units][cap]
};

// One row's settings.
struct Setting {
    double c;  // log2(e) / temperature
    uint32_t k;
    double p, min_p;
    bool top_p_on, min_p_on;
    __device__ __forceinline__ Setting(const SampleArgs& a, int b)
    {
        const float t = fminf(a.temperature_rows ? a.temperature_rows[b] : a.temperature, FLT_MAX);
        const int64_t kk = a.top_k_rows ? (int64_t)a.top_k_rows[b] : a.top_k;
        const float pp = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
        const float mm = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
        // (NaN: greedy; fminf drops it, so the setting itself is asked)
        const bool greedy = !((a.temperature_rows ? a.temperature_rows[b] : a.temperature) > 0.0f);
        c = greedy ? LOG2E_F64 : LOG2E_F64 / (double)t;
        k = greedy ? 1u : kk > 0 && kk < a.vocab ? (uint32_t)kk : 0u;
        top_p_on = pp < 1.0f;
        p = (double)fmaxf(pp, 0.0f);
        min_p_on = !(mm <= 0.0f);
        min_p = (double)fminf(mm, 1.0f);  // (NaN: 1)
    }
    __device__ __forceinline__ bool whole_sum() const { return k == 0 && (top_p_on || !min_p_on); }
    __device__ __forceinline__ bool border() const { return k > 0 || top_p_on || min_p_on; }
};

// The blocks of a row: 16 aligned bytes each, the first and last possibly
// reaching over its ends.
template <int LT>
struct Row {
    static constexpr int VEC = LT == VQ2_DT_F32 ? 4 : 8;
    const void* p;
    int64_t start;  // element of the row's first column
    int off;        // columns of block 0 before it
    int vocab, blocks;
    __device__ __forceinline__ Row(const SampleArgs& a, int b) : p(a.logits), start(b * a.stride), vocab(a.vocab)
    {
        const uintptr_t at = (uintptr_t)a.logits + start * (16 / VEC);
        off = (int)(at & 15) / (16 / VEC);
        blocks = (vocab + off + VEC - 1) / VEC;
    }
    __device__ __forceinline__ int column(int block) const { return block * VEC - off; }
    // The columns of a block, -inf where it reaches over the row's ends; an
    // infinite logit becomes the largest finite one (no difference of
    // infinities), NaN stays
    __device__ __forceinline__ void load(int block, float (&v)[VEC]) const
    {
        const int c0 = column(block);
        if (c0 >= 0 && c0 + VEC <= vocab) {
            if constexpr (LT == VQ2_DT_F32) {
                const u32x4 w = *(const u32x4*)((const float*)p + start + c0);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = __uint_as_float(w[i]);
            } else {
                const u32x4 w = *(const u32x4*)((const uint16_t*)p + start + c0);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t h = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
                    v[i] = LT == VQ2_DT_F16 ? f16_bits_to_f32((uint16_t)h) : bf16_bits_to_f32(h);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                v[i] = c0 + i >= 0 && c0 + i < vocab ? ld_t<LT>(p, start + c0 + i) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = v[i] == INFINITY ? FLT_MAX : v[i];
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

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// ------------------------------------------------------------ first launch
template <int LT>
__global__ void __launch_bounds__(NT) sample_stats_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.arrivals[b] = 0;
    const int unit = blockIdx.x * NW + (threadIdx.x >> 6);
    if (unit >= a.units) return;
    const Setting s(a, b);
    const Row<LT> row(a, b);
    const int end = min(row.blocks, (unit + 1) * a.unit_blocks);
    float m = -INFINITY;
    double sum = 0.0;
    if (s.whole_sum()) {
        // sum of exp((l - ref) / temperature), ref one of the lane's logits:
        // 64 bits hold weights of 2^1000, so it moves only where one is close
        float ref = -INFINITY;
        for (int i = unit * a.unit_blocks + lane; i < end; i += 64) {
            float v[VEC];
            row.load(i, v);
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
        }
        const float um = wave_max_all(m);
        sum = wave_sum_f64(sum * exp2_f64(((double)ref - (double)um) * s.c));
    } else {
#pragma unroll 4
        for (int i = unit * a.unit_blocks + lane; i < end; i += 64) {
            float v[VEC];
            row.load(i, v);
#pragma unroll
            for (int j = 0; j < VEC; j++) m = fmaxf(m, v[j]);
        }
    }
    const int64_t at = (int64_t)b * a.units + unit;
    if (s.k > 1) {
        float g = m;
        if (a.fine == 4) {
            g = fmaxf(g, dpp_xor1(g));
            g = fmaxf(g, dpp_xor2(g));
            g = fmaxf(g, dpp_half_mirror(g));
            g = fmaxf(g, dpp_row_mirror(g));
            if ((lane & 15) == 0) a.fine_max[at * 4 + lane / 16] = g;
        } else {
            a.fine_max[at * 64 + lane] = g;
        }
    }
    m = wave_max_all(m);
    if (lane == 0) {
        a.unit_max[at] = m;
        a.unit_sum[at] = sum;
    }
}

// ----------------------------------------------------------- second launch
struct Shared {
    uint64_t list[LIST];     // the row's entries in column order
    uint64_t amount[NT];     // a histogram's sums
    uint32_t count[NT];      // and its entries
    uint32_t first[NT + 1];  // entries of the list before a unit's
    uint64_t wave64[NW + 2];
    double wave_d[NW + 2];
    uint32_t small_n;
};

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, int lane)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// Inclusive running sum over the workgroup; total in every thread.
__device__ __forceinline__ uint64_t block_scan(Shared& sh, uint64_t v, uint64_t& total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = wave_scan_u64(v, lane);
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

__device__ __forceinline__ float block_max(Shared& sh, float v)
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

__device__ __forceinline__ int block_min(Shared& sh, int v)
{
    for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave64[threadIdx.x >> 6] = (uint64_t)(uint32_t)v;
    __syncthreads();
    int m = (int)(uint32_t)sh.wave64[0];
#pragma unroll
    for (int i = 1; i < NW; i++) m = min(m, (int)(uint32_t)sh.wave64[i]);
    return m;
}

// A row's weights of 64 bits and of whole numbers.
struct Weigher {
    float max;
    double c;
    __device__ __forceinline__ double operator()(float l) const
    {
        const double d = ((double)l - (double)max) * c;
        return d > -999.0 ? exp2_f64(d) : 0.0;  // (NaN: 0)
    }
};

// The entries that a border is sought among: the list in LDS, ...
struct ListSource {
    const uint64_t* list;
    int n;
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        for (int i = threadIdx.x; i < n; i += NT) f(list[i]);
    }
    // the kept weight of thread t's piece of the list, pieces in column order
    template <class F>
    __device__ __forceinline__ uint64_t piece(int t, F kept) const
    {
        const int per = (n + NT - 1) / NT;
        uint64_t s = 0;
        for (int i = t * per; i < min(n, (t + 1) * per); i++) s += kept(list[i]);
        return s;
    }
    // the entry of that piece at which the running sum from `run` on exceeds target
    template <class F>
    __device__ __forceinline__ uint64_t find(int t, uint64_t run, uint64_t target, F kept) const
    {
        const int per = (n + NT - 1) / NT;
        for (int i = t * per; i < min(n, (t + 1) * per); i++) {
            run += kept(list[i]);
            if (run > target) return list[i];
        }
        return 0;
    }
};

// ... or the row itself, its entries from `cut` on.
template <int LT>
struct RowSource {
    const Row<LT>& row;
    float cut;
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        for (int i = threadIdx.x; i < row.blocks; i += NT) block(i, f);
    }
    template <class F>
    __device__ __forceinline__ void block(int i, F f) const
    {
        constexpr int VEC = Row<LT>::VEC;
        float v[VEC];
        row.load(i, v);
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (v[j] >= cut) f(order_key(v[j], row.column(i) + j));
    }
    template <class F>
    __device__ __forceinline__ uint64_t piece(int t, F kept) const
    {
        const int per = (row.blocks + NT - 1) / NT;
        uint64_t s = 0;
        for (int i = t * per; i < min(row.blocks, (t + 1) * per); i++) block(i, [&](uint64_t key) { s += kept(key); });
        return s;
    }
    template <class F>
    __device__ __forceinline__ uint64_t find(int t, uint64_t run, uint64_t target, F kept) const
    {
        const int per = (row.blocks + NT - 1) / NT;
        uint64_t found = 0;
        for (int i = t * per; i < min(row.blocks, (t + 1) * per); i++)
            block(i, [&](uint64_t key) {
                const uint64_t before = run;
                run += kept(key);
                if (before <= target && run > target) found = key;
            });
        return found;
    }
};

// The border of the entries in [lo, hi]: the key of the last one that stays
// when an entry stays while the amounts before it are below `limit` (>= 1).
// Each round is a histogram of the keys over 1024 equal ranges (a suffix sum
// by the workgroup's threads finds the range that the limit falls into); keys
// differ, so the rounds end.  lo if all stay.
template <class Source, class F>
__device__ uint64_t find_border(Shared& sh, const Source& src, uint64_t lo, uint64_t hi, uint64_t limit, F amount)
{
    const int tid = threadIdx.x;
    uint64_t before = 0;
    for (;;) {
        // ranges of 2^shift keys, range 0 the highest
        const uint64_t span = hi - lo;
        const int shift = span < NT ? 0 : 64 - __clzll(span) - 10;
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
        const uint64_t run = before + block_scan(sh, mine, all);
        if (before + all < limit) return lo;  // (the first round only)
        if (run >= limit && run - mine < limit) {
            sh.wave64[NW] = (uint64_t)tid;
            sh.wave64[NW + 1] = run - mine;
        }
        __syncthreads();
        const int r = (int)(sh.wave64[NW] & (NT - 1));
        before = sh.wave64[NW + 1];
        const uint32_t m = min(sh.count[r], (uint32_t)NT);
        hi -= (uint64_t)r << shift;
        const uint64_t width = shift >= 64 ? ~0ull : (1ull << shift) - 1;
        lo = hi - lo < width ? lo : hi - width;
        if (m > DIRECT && shift > 0) continue;
        // rank the m entries directly
        if (tid == 0) sh.small_n = 0;
        __syncthreads();
        src.each([&](uint64_t key) {
            if (key >= lo && key <= hi) sh.amount[atomicAdd(&sh.small_n, 1u) & (NT - 1)] = key;
        });
        __syncthreads();
        uint64_t last = ~0ull;
        if (tid < (int)m) {
            const uint64_t key = sh.amount[tid];
            uint64_t above = before;
            for (int j = 0; j < (int)m; j++) {
                const uint64_t o = sh.amount[j];
                if (o > key) above += amount(o);
            }
            if (above < limit) last = key;
        }
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor(last, off);
            last = o < last ? o : last;
        }
        __syncthreads();
        if ((tid & 63) == 0) sh.wave64[tid >> 6] = last;
        __syncthreads();
        for (int i = 0; i < NW; i++) last = sh.wave64[i] < last ? sh.wave64[i] : last;
        return last;
    }
}

// Border and draw among the entries of a source.
template <class Source>
__device__ void finish(Shared& sh, const SampleArgs& a, const Setting& s, const Weigher& weigh, const Source& src, float cut,
                       double z, int b)
{
    auto mass = [&](uint64_t key) { return fixed(weigh(key_logit(key))); };
    uint64_t lo = order_key(cut, 0) & ~0xFFFFFFFFull;
    const uint64_t hi = order_key(weigh.max, 0) | 0xFFFFFFFFull;
    if (s.k > 0) lo = find_border(sh, src, lo, hi, (uint64_t)s.k, [](uint64_t) { return 1ull; });
    uint64_t total;
    if (s.top_p_on) {
        double all = z * UNIT;
        if (s.k > 0) {
            uint64_t part = 0;
            src.each([&](uint64_t key) { part += key >= lo ? mass(key) : 0; });
            block_scan(sh, part, total);
            all = (double)total;
        }
        const double limit = ceil(s.p * all);
        lo = find_border(sh, src, lo, hi, limit > 1.0 ? (uint64_t)limit : 1, mass);
    }
    auto kept = [&](uint64_t key) -> uint64_t {
        if (key < lo) return 0;
        const double w = weigh(key_logit(key));
        return !s.min_p_on || w >= s.min_p ? fixed(w) : 0;
    };
    const uint64_t mine = src.piece(threadIdx.x, kept);
    const uint64_t run = block_scan(sh, mine, total);
    const double at = fmin(fmax((double)a.u[b], 0.0), 1.0) * (double)total;
    uint64_t target = (uint64_t)at;
    if (target >= total) target = total - 1;
    if (run > target && run - mine <= target) {
        const uint64_t key = src.find((int)threadIdx.x, run - mine, target, kept);
        const double d = ((double)key_logit(key) - (double)weigh.max) * s.c;
        a.out_idx[b] = key_column(key);
        a.out_logprob[b] = (float)(d / LOG2E_F64 - log((double)total / UNIT));
    }
}

template <int LT>
__global__ void __launch_bounds__(NT) sample_pick_kernel(SampleArgs a)
{
    constexpr int VEC = Row<LT>::VEC;
    __shared__ Shared sh;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Setting s(a, b);
    const bool first = s.k == 1 || !s.border();  // one workgroup is enough
    if (first && blockIdx.x > 0) return;
    const Row<LT> row(a, b);
    const int64_t units0 = (int64_t)b * a.units;
    const float um = tid < a.units ? a.unit_max[units0 + tid] : -INFINITY;
    const float m = block_max(sh, um);
    if (m == -INFINITY) {
        if (blockIdx.x == 0 && tid == 0) {
            a.out_idx[b] = -1;
            a.out_logprob[b] = NAN;
        }
        return;
    }
    const Weigher weigh{m, s.c};
    if (s.k == 1) {  // the first maximum
        const int unit = block_min(sh, um == m ? tid : MAX_UNITS);
        const int end = min(row.blocks, (unit + 1) * a.unit_blocks);
        int col = 0x7FFFFFFF;
        for (int i = unit * a.unit_blocks + tid; i < end; i += NT) {
            float v[VEC];
            row.load(i, v);
#pragma unroll
            for (int j = VEC - 1; j >= 0; j--)
                if (v[j] == m) col = min(col, row.column(i) + j);
        }
        col = block_min(sh, col);
        if (tid == 0) {
            a.out_idx[b] = col;
            a.out_logprob[b] = 0.0f;
        }
        return;
    }
    double z = 0.0;
    if (s.whole_sum()) {
        // running sums of the units' weights; a thread's sum ends where the next one's begins
        double v = tid < a.units ? a.unit_sum[units0 + tid] * exp2_f64(((double)um - (double)m) * s.c) : 0.0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(v, off);
            if (lane >= off) v += o;
        }
        __syncthreads();
        if (lane == 63) sh.wave_d[wave] = v;
        __syncthreads();
        double before = 0.0;
        for (int i = 0; i < wave; i++) before += sh.wave_d[i];
        double* const ends = (double*)sh.amount;
        ends[tid] = before + v;
        __syncthreads();
        z = ends[NT - 1];
        if (first) {
            const double target = fmin(fmax((double)a.u[b], 0.0), 1.0) * z;
            // the unit, then the column, whose running sum is the first above
            // the target (the last with a weight, if rounding leaves none)
            const bool live = tid < a.units && um > -INFINITY && ends[tid] > (tid ? ends[tid - 1] : 0.0);
            int unit = block_min(sh, live && ends[tid] > target ? tid : MAX_UNITS);
            if (unit == MAX_UNITS) unit = MAX_UNITS - 1 - block_min(sh, live ? MAX_UNITS - 1 - tid : MAX_UNITS - 1);
            const double base = unit ? ends[unit - 1] : 0.0;
            const int b0 = unit * a.unit_blocks, end = min(row.blocks, b0 + a.unit_blocks);
            const int per = (a.unit_blocks + NT - 1) / NT;
            double mine = 0.0;
            float v4[VEC];
            for (int i = b0 + tid * per; i < min(end, b0 + (tid + 1) * per); i++) {
                row.load(i, v4);
#pragma unroll
                for (int j = 0; j < VEC; j++) mine += weigh(v4[j]);
            }
            double run = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const double o = __shfl_up(run, off);
                if (lane >= off) run += o;
            }
            __syncthreads();
            if (lane == 63) sh.wave_d[wave] = run;
            __syncthreads();
            before = base;
            for (int i = 0; i < wave; i++) before += sh.wave_d[i];
            ends[tid] = before + run;
            __syncthreads();
            int t = block_min(sh, mine > 0.0 && ends[tid] > target ? tid : NT);
            if (t == NT) t = NT - 1 - block_min(sh, mine > 0.0 ? NT - 1 - tid : NT - 1);
            if (tid == t) {
                double at = t ? ends[t - 1] : base;
                int col = 0;
                float l = m;
                bool done = false;
                for (int i = b0 + tid * per; i < min(end, b0 + (tid + 1) * per); i++) {
                    row.load(i, v4);
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const double w = weigh(v4[j]);
                        at += w;
                        if (!done && w > 0.0) {
                            col = row.column(i) + j;
                            l = v4[j];
                            done = at > target;
                        }
                    }
                }
                a.out_idx[b] = col;
                a.out_logprob[b] = (float)(((double)l - (double)m) * s.c / LOG2E_F64 - log(z));
            }
            return;
        }
    }
    // the logit from which on entries may stay (rounded down, by more than the
    // arithmetic here is off)
    double low = (double)m - 45.0 / s.c;  // w < 2^-45
    if (s.k == 0) {
        if (s.top_p_on) low = fmax(low, (double)m + log2((1.0 - s.p) * 0.999 * z / (double)a.vocab) / s.c);
        if (s.min_p_on) low = fmax(low, (double)m + log2(s.min_p * 0.999) / s.c);
    } else {
        if (s.min_p_on && !s.top_p_on) low = fmax(low, (double)m + log2(s.min_p * 0.999) / s.c);
        // the range of 1024 between the lowest and the highest maximum that
        // the k-th largest one falls into; more groups than k are needed
        const bool coarse = s.k * 2 <= (uint32_t)a.units;
        const int groups = coarse ? a.units : a.units * a.fine;
        if (s.k * 5 <= (uint32_t)groups * 4) {
            const float* const g = coarse ? a.unit_max + units0 : a.fine_max + units0 * a.fine;
            float least = INFINITY;
            for (int i = tid; i < groups; i += NT) least = fminf(least, fmaxf(g[i], (float)fmax(low, (double)-FLT_MAX)));
            least = -block_max(sh, -least);
            const uint32_t top = (uint32_t)(order_key(m, 0) >> 32), bottom = (uint32_t)(order_key(least, 0) >> 32);
            const int shift = top - bottom < NT ? 0 : 32 - __clz(top - bottom) - 10;
            __syncthreads();
            sh.count[tid] = 0;
            __syncthreads();
            for (int i = tid; i < groups; i += NT) {
                const uint32_t key = (uint32_t)(order_key(g[i], 0) >> 32);
                if (g[i] >= least) atomicAdd(&sh.count[(top - key) >> shift], 1u);
            }
            __syncthreads();
            uint64_t all;
            const uint64_t mine = sh.count[tid], run = block_scan(sh, mine, all);
            if (tid == 0) sh.wave64[NW] = NT;
            __syncthreads();
            if (run >= s.k && run - mine < s.k) sh.wave64[NW] = (uint64_t)tid;
            __syncthreads();
            const int r = (int)sh.wave64[NW];
            if (r < NT) {  // the lowest key of range r
                const uint64_t down = (((uint64_t)r + 1) << shift) - 1;
                const uint32_t key = down < top - bottom ? top - (uint32_t)down : bottom;
                low = fmax(low, (double)key_logit((uint64_t)key << 32));
            }
        }
    }
    const double slack = fabs((double)m) * 1e-6 + fabs(low) * 1e-6;
    const float cut = (float)fmax(low - slack, (double)-FLT_MAX);

    // this wave's unit, in column order
    const int unit = blockIdx.x * NW + wave;
    if (unit < a.units) {
        uint64_t* const list = a.list + (units0 + unit) * a.cap;
        int n = 0;
        const int b0 = unit * a.unit_blocks;
        for (int i0 = 0; i0 < a.unit_blocks; i0 += 64) {
            const int i = b0 + i0 + lane;
            float v[VEC];
            int mine = 0;
            if (i < row.blocks) {
                row.load(i, v);
#pragma unroll
                for (int j = 0; j < VEC; j++) mine += v[j] >= cut;
            }
            if (__ballot(mine > 0) == 0) continue;
            int end = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(end, off);
                if (lane >= off) end += o;
            }
            int at = n + end - mine;
            if (mine > 0) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (v[j] >= cut) {
                        if (at < a.cap)
                            __hip_atomic_store(list + at, order_key(v[j], row.column(i) + j), __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT);
                        at++;
                    }
            }
            n += __shfl(end, 63);
        }
        if (lane == 0)
            __hip_atomic_store(a.list_len + units0 + unit, (uint32_t)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!arrive_last(a.arrivals + b, gridDim.x)) return;

    // the row's last workgroup: the list to LDS
    uint32_t len = tid < a.units ? __hip_atomic_load(a.list_len + units0 + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    uint64_t all;
    const uint64_t over = len > (uint32_t)a.cap ? 1ull << 40 : 0;
    const uint64_t run = block_scan(sh, len | over, all);
    if (all <= LIST) {
        sh.first[tid + 1] = (uint32_t)run;
        if (tid == 0) sh.first[0] = 0;
        __syncthreads();
        const int n = (int)all;
        for (int i = tid; i < n; i += NT) {
            int at = 0;  // the unit: first[at] <= i < first[at + 1]
#pragma unroll
            for (int step = NT / 2; step > 0; step >>= 1)
                if (sh.first[at + step] <= (uint32_t)i) at += step;
            sh.list[i] = __hip_atomic_load(a.list + (units0 + at) * a.cap + (i - sh.first[at]), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        finish(sh, a, s, weigh, ListSource{sh.list, n}, cut, z, b);
    } else {
        finish(sh, a, s, weigh, RowSource<LT>{row, cut}, cut, z, b);
    }
}

// How a call is cut: units of at least 64 blocks (one load a lane), longer
// ones where the rows alone make 1024 workgroups of 16 units.
struct Plan {
    int units, unit_blocks, fine, cap;
    size_t arrivals, unit_sum, unit_max, fine_max, list_len, list, bytes;
};

Plan make_plan(int64_t rows, int64_t vocab, int vec)
{
    Plan p;
    const int64_t blocks = (vocab + 2 * vec - 2) / vec;  // (any alignment)
    int64_t per = (blocks * rows + 1024 * NW - 1) / (1024 * NW);
    per = per > (blocks + MAX_UNITS - 1) / MAX_UNITS ? per : (blocks + MAX_UNITS - 1) / MAX_UNITS;
    per = per > (blocks + NW - 1) / NW ? (blocks + NW - 1) / NW : per;
    p.unit_blocks = (int)((per + 63) / 64 * 64);
    p.units = (int)((blocks + p.unit_blocks - 1) / p.unit_blocks);
    p.fine = p.units >= 512 ? 4 : 64;
    const int entries = p.unit_blocks * vec;
    p.cap = entries <= 512 ? entries : entries / 4 > 512 ? entries / 4 : 512;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t r = at;
        at += (n + 255) / 256 * 256;
        return r;
    };
    const size_t n = (size_t)rows * p.units;
    p.arrivals = take(rows * 4);
    p.unit_sum = take(n * 8);
    p.unit_max = take(n * 4);
    p.fine_max = take(n * p.fine * 4);
    p.list_len = take(n * 4);
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
                       (uint32_t*)(ws + p.arrivals), (double*)(ws + p.unit_sum), (float*)(ws + p.unit_max),
                       (float*)(ws + p.fine_max), (uint32_t*)(ws + p.list_len), (uint64_t*)(ws + p.list)};
    hipStream_t st = (hipStream_t)c.stream;
    const dim3 grid((unsigned)((p.units + NW - 1) / NW), (unsigned)c.rows), block(NT);
    hipLaunchKernelGGL(sample_stats_kernel<LT>, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_pick_kernel<LT>, grid, block, 0, st, a);
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
