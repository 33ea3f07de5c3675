// vq2_panel.hip -- many-row products of packed matrices on the matrix cores,
// with what follows them in their epilogues, and the gradients through the
// frozen codes:
//
//   gated block   act = f(s_g Wg x) (s_u Wu x), and its backward pass
//   head's loss   lse_t = log sum_v exp(s_v W_v x_t), loss = lse - logit of
//                 the target, and its backward pass
//   product       dx = (s dy) W and ds_v = sum_t dy_tv W_v x_t
//
// A call packs the token rows into a panel (vq2_panel.hpp), and takes the
// matrix in pieces of rows: a piece's codes are turned into panels of fp16
// weights in a workspace (rows of n values; for a gradient also columns of
// piece values), which the products then read.  Logits and their gradients
// exist for one piece at a time.
//
// Rounding.  A token row is held in fp16 under a power of two of its own (11
// bits: exact for fp16, bf16 and 8-bit rows but for values 2^-28 below the
// row's largest).  A weight is the fp32 sum of its stages' centroids, exact
// in fp16 for one stage of fp16 codebooks; otherwise it is rounded to fp16
// where only bf16 results depend on it (half a step is 2^-11 of a weight,
// against 2^-8 of the result), and held as two fp16 parts, multiplied one
// after the other, where an fp16 or fp32 result does.  Row scales stay outside,
// in fp32.  A gradient is rounded to fp16 once between its two products (2^-11
// of each term; what comes of it has 16 bits), under powers of two that hold the
// largest: of a token's upstream values, of the row scales, and in the block's
// backward pass of |u f'(g)| and |f(g)|, which a bound on the products holds
// (BlockBound).  Everything else is fp32.
#include <algorithm>
#include <mutex>

#include "vq2_internal.hpp"
#include "vq2_panel.hpp"

namespace vq2 {

namespace {

// ------------------------------------------------------------- conversions
constexpr float NEG_INF = -__builtin_inff();

// 2^e, |e| <= 126
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// exponent e with |v| < 2^(e+1); 0 for 0, infinities and NaN
__device__ __forceinline__ int exponent_of(float v)
{
    const int b = (int)(__float_as_uint(v) >> 23 & 0xFF);
    return b == 0xFF || (__float_as_uint(v) & 0x7FFFFFFFu) == 0 ? 0 : b - 127;
}

// Exponent of a power of two not below any row scale, from the largest
// magnitudes of the prologue's workgroups; bounded so that 2^(15 - e) and 2^e
// are normal numbers.  Called by whole waves.
struct RowTop {
    const float* part;
    int n;
};
__device__ __forceinline__ int scale_exponent(const RowTop& t)
{
    float m = 0.0f;
    for (int i = threadIdx.x & 63; i < t.n; i += 64) m = fmaxf(m, t.part[i]);
    const int b = (int)(__float_as_uint(wave_max_all(m)) >> 23);
    return b == 0xFF ? 0 : min(max(b - 126, -100), 100);
}

// The block's backward pass: exponent of a power of two above 1.13 |u| and 1.13 |g| of a
// token, which bounds |u f'(g)| and |f(g)|, from the largest of its row, of the
// codebooks and of the scales, and the row's length.  Of random rows the largest of them
// is some 2^10 smaller, which fp16's 30 binades hold.
struct BlockBound {
    RowTop amax, books;
    const float* fac;  // of the token rows: |x| < 2^14 fac
    int bits;          // 14 + log2(n), rounded up, + 1, + 1 for a second stage
    // the part that tokens share; called by whole waves
    __device__ __forceinline__ int common() const
    {
        float m = 0.0f;
        for (int i = threadIdx.x & 63; i < books.n; i += 64) m = fmaxf(m, books.part[i]);
        return bits + scale_exponent(amax) + exponent_of(wave_max_all(m)) + 1;
    }
    __device__ __forceinline__ int of(int common, int t) const { return common + exponent_of(fac[t]); }
};
// 2^e as far as it is a normal number
__device__ __forceinline__ float pow2_near(int e) { return pow2(min(max(e, -126), 126)); }

// over the four lanes that hold a token's rows
__device__ __forceinline__ float max_rows(float v)
{
    v = fmaxf(v, swz_xor16(v));
    return fmaxf(v, xor32(v));
}
__device__ __forceinline__ float sum_rows(float v)
{
    v += swz_xor16(v);
    return v + xor32(v);
}

// ------------------------------------------------------------ packed rows
// Rows of the matrices in tiles of 16: one matrix in order; two (gate, up)
// in turn, so that a wave finds both products of a row in its registers.
struct PanelMat {
    const int16_t* i0;
    const void* i1;
    const void* scale;
};
struct MatArgs {
    PanelMat m[2];
    int nmat;
    int64_t rows;  // of each
    int ng;        // groups of 8 values
    int s_dt;
    const void* cb0;
    const void* cb1;
};
__device__ __forceinline__ int64_t mat_row(const MatArgs& a, int64_t tile, int r, int& mat)
{
    mat = a.nmat == 2 ? (int)(tile & 1) : 0;
    return (a.nmat == 2 ? tile >> 1 : tile) * 16 + r;
}

// What a wave finds of two row tiles in its registers is the operand of the
// next product: lane (q, t) holds rows 4 q .. + 3 of both, 8 values, and that is
// its chunk q of a k tile of 32 rows as long as the columns' panel has the
// same order (value m of chunk q: row 16 (m / 4) + 4 q + m % 4).  So a
// gradient is stored as it is made, a KiB a tile.

// -------------------------------------------------------------- prologue
// One launch: token rows, upstream rows' factors, row scales.
struct PackArgs {
    const void* x;
    int x_dt;
    int tokens, n;  // rows past the last token are zeros
    const float* x_scale;
    const int64_t* target;  // or null: rows whose target is `ignore` are zeros, too
    int64_t ignore;
    half8_t* panel;     // [tiles][n / 32][64]
    float* fac;         // a product of the panel times fac[t] is one of the row
    int tiles;          // 0: no rows to pack
};

// One workgroup a tile of 16 rows, its 16 waves a share of the k tiles each:
// the rows' largest magnitudes, then fp16 under a power of two that brings
// them into [2^13, 2^14).  Rows of up to 4096 values stay in registers in
// between (4096 rows of 2048: 21 us with 4 waves that read twice).
constexpr int PK_WAVES = 16, PK_HELD = 8;
template <int DT>
__device__ __forceinline__ void pack_rows(const PackArgs& a, int tile, float (*s_m)[16])
{
    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6, row = tile * 16 + (lane & 15), q = lane >> 4, kt = a.n / 32;
    const int per = (kt + PK_WAVES - 1) / PK_WAVES, k0 = wave * per, k1 = min(k0 + per, kt);
    const bool live = row < a.tokens && !(a.target && a.target[row] == a.ignore), held = per <= PK_HELD;
    const int64_t at = (int64_t)row * a.n + q * 8;
    Eight x[PK_HELD];
    float m = 0.0f;
    if (held) {
#pragma unroll
        for (int i = 0; i < PK_HELD; i++)
            if (live && k0 + i < k1) x[i] = load8(a.x, DT, at + (k0 + i) * 32);
            else
#pragma unroll
                for (int k = 0; k < 8; k++) x[i].v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < PK_HELD; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(x[i].v[k]));
    } else if (live) {
        for (int k = k0; k < k1; k++) {
            const Eight e = load8(a.x, DT, at + k * 32);
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(e.v[j]));
        }
    }
    m = max_rows(m);
    if (q == 0) s_m[wave][lane & 15] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PK_WAVES; w++) m = fmaxf(m, s_m[w][lane & 15]);
    // (8-bit values are exact as they are)
    const int e = DT <= VQ2_DT_BF16 && m > 0.0f ? min(max(exponent_of(m) - 13, -110), 110) : 0;
    if (tid < 16) a.fac[row] = live ? pow2(e) * (a.x_scale ? a.x_scale[row] : 1.0f) : 0.0f;
    const float f = pow2(-e);
    half8_t* out = a.panel + (int64_t)tile * kt * 64 + lane;
    if (held) {
#pragma unroll
        for (int i = 0; i < PK_HELD; i++) {
            if (k0 + i >= k1) break;
            half8_t h;
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = (_Float16)(x[i].v[j] * f);
            out[(k0 + i) * 64] = h;
        }
    } else {
        for (int k = k0; k < k1; k++) {
            half8_t h = {0, 0, 0, 0, 0, 0, 0, 0};
            if (live) {
                const Eight v = load8(a.x, DT, at + k * 32);
#pragma unroll
                for (int j = 0; j < 8; j++) h[j] = (_Float16)(v.v[j] * f);
            }
            out[k * 64] = h;
        }
    }
}

struct DyMaxArgs {
    const void* dy;
    int dy_dt, tokens, vec;  // vec: rows a multiple of 8, 16-byte aligned
    int64_t rows;
    float* dfac;  // [tp]: 2^-e, which brings the row's largest into [2^14, 2^15)
    int groups;   // of 16 rows
};
// a wave a row
template <int DT>
__device__ __forceinline__ void dy_max(const DyMaxArgs& a, int group)
{
    const int lane = threadIdx.x & 63, t = group * PK_WAVES + (threadIdx.x >> 6);
    float m = 0.0f;
    if (t < a.tokens) {
        const int64_t at = t * a.rows;
        if (a.vec) {
#pragma unroll 4
            for (int64_t i = lane * 8; i < a.rows; i += 512) {
                const Eight e = load8(a.dy, DT, at + i);
#pragma unroll
                for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(e.v[k]));
            }
        } else {
#pragma unroll 4
            for (int64_t i = lane; i < a.rows; i += 64) m = fmaxf(m, fabsf(load_as_f32(a.dy, DT, at + i)));
        }
    }
    m = wave_max_all(m);
    const int e = m > 0.0f ? min(max(exponent_of(m) - 14, -110), 110) : 0;
    if (lane == 0) a.dfac[t] = pow2(-e);
}

struct PrepArgs {
    MatArgs m;
    float rs;
    int64_t places;  // 16 * tiles
    float* sc;       // scale * rs of each place, 0 past the last row
    float* top;      // largest magnitude of each workgroup's
    int groups;      // of PREP_ROWS places
};
constexpr int PREP_ROWS = 4 * 64 * PK_WAVES;
__device__ __forceinline__ void prep_scales(const PrepArgs& a, int group, float* s_top)
{
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int64_t p = (int64_t)group * PREP_ROWS + k * 64 * PK_WAVES + threadIdx.x;
        if (p >= a.places) continue;
        int mat;
        const int64_t row = mat_row(a.m, p >> 4, (int)(p & 15), mat);
        const float v = row < a.m.rows ? load_as_f32(a.m.m[mat].scale, a.m.s_dt, row) * a.rs : 0.0f;
        a.sc[p] = v;
        m = fmaxf(m, fabsf(v));
    }
    m = wave_max_all(m);
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 0; k < PK_WAVES; k++) m = fmaxf(m, s_top[k]);
    a.top[group] = m;
}

// The codebooks' largest magnitudes, BOOK_VALUES values a workgroup.
struct BookArgs {
    const void* cb[2];
    int cb_dt, n0;          // workgroups of the first
    int64_t values[2];      // multiples of 8
    float* top;             // of each workgroup
    int groups;
};
constexpr int BOOK_VALUES = 8 * 64 * PK_WAVES;
template <int CBT>
__device__ __forceinline__ void book_max(const BookArgs& a, int group, float* s_top)
{
    const int k = group >= a.n0;
    const int64_t at = (int64_t)(group - (k ? a.n0 : 0)) * BOOK_VALUES + threadIdx.x * 8;
    float m = 0.0f;
    if (at < a.values[k]) {
        const Eight e = load8(a.cb[k], CBT, at);
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(e.v[j]));
    }
    m = wave_max_all(m);
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 0; w < PK_WAVES; w++) m = fmaxf(m, s_top[w]);
    a.top[group] = m;
}

struct PrologueArgs {
    PackArgs pack;
    DyMaxArgs dy;
    PrepArgs prep;
    BookArgs book;
};
__global__ void __launch_bounds__(64 * PK_WAVES) prologue_kernel(const PrologueArgs a)
{
    __shared__ float s_m[PK_WAVES][16];
    int b = blockIdx.x;
    // (types apart: behind a branch on the type every load is waited for)
    if (b < a.pack.tiles) {
        if (a.pack.x_dt == VQ2_DT_F16) return pack_rows<VQ2_DT_F16>(a.pack, b, s_m);
        if (a.pack.x_dt == VQ2_DT_BF16) return pack_rows<VQ2_DT_BF16>(a.pack, b, s_m);
        if (a.pack.x_dt == VQ2_DT_I8) return pack_rows<VQ2_DT_I8>(a.pack, b, s_m);
        return pack_rows<VQ2_DT_E4M3>(a.pack, b, s_m);
    }
    b -= a.pack.tiles;
    if (b < a.dy.groups) {
        if (a.dy.dy_dt == VQ2_DT_F16) return dy_max<VQ2_DT_F16>(a.dy, b);
        if (a.dy.dy_dt == VQ2_DT_BF16) return dy_max<VQ2_DT_BF16>(a.dy, b);
        return dy_max<VQ2_DT_F32>(a.dy, b);
    }
    b -= a.dy.groups;
    if (b < a.prep.groups) return prep_scales(a.prep, b, s_m[0]);
    b -= a.prep.groups;
    if (a.book.cb_dt == VQ2_DT_F16) return book_max<VQ2_DT_F16>(a.book, b, s_m[0]);
    if (a.book.cb_dt == VQ2_DT_BF16) return book_max<VQ2_DT_BF16>(a.book, b, s_m[0]);
    book_max<VQ2_DT_F32>(a.book, b, s_m[0]);
}

template <int CBT>
__device__ __forceinline__ void centroid_f32(const void* cb, uint32_t c, float (&w)[8])
{
    const Eight e = load8(cb, CBT, (int64_t)c * 8);
#pragma unroll
    for (int k = 0; k < 8; k++) w[k] = e.v[k];
}

// fp16 weight of a code pair; PARTS == 2: what its rounding leaves, too
template <int CBT, int S2, int PARTS>
__device__ __forceinline__ void weight_of(const MatArgs& a, uint32_t c0, uint32_t c1, half8_t& hi, half8_t& lo)
{
    if constexpr (CBT == VQ2_DT_F16 && S2 == VQ2_S2_NONE) {
        hi = ((const half8_t*)a.cb0)[c0];
    } else {
        float w[8], u[8];
        centroid_f32<CBT>(a.cb0, c0, w);
        if constexpr (S2 != VQ2_S2_NONE) {
            centroid_f32<CBT>(a.cb1, c1, u);
#pragma unroll
            for (int k = 0; k < 8; k++) w[k] += u[k];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            hi[k] = (_Float16)w[k];
            if constexpr (PARTS == 2) lo[k] = (_Float16)(w[k] - (float)hi[k]);
        }
    }
}

template <int S2>
__device__ __forceinline__ uint32_t code1(const void* i1, int64_t i)
{
    if constexpr (S2 == VQ2_S2_U8) return ((const uint8_t*)i1)[i];
    if constexpr (S2 == VQ2_S2_U16) return ((const uint16_t*)i1)[i];
    return 0;
}

struct DequantArgs {
    MatArgs m;
    int64_t tile0;  // the piece's first tile
    half8_t* w;     // [tiles][PARTS * ng / 4][64]
    half8_t* wt;    // [columns / 16][parts * tiles / 2][64], or null
    int vkt;        // tiles / 2
    int vec;        // planes of 16-byte aligned rows
};

// 8 codes of consecutive groups as words of two 16-bit codes (uint8 planes:
// of four)
template <int B>
__device__ __forceinline__ u32x4 codes8(const void* p, int64_t i)
{
    if constexpr (B == 2) return *(const u32x4*)((const uint16_t*)p + i);
    const u32x2 u = *(const u32x2*)((const uint8_t*)p + i);
    return u32x4{u.x, u.y, 0, 0};
}
// lane (row, q)'s code of k tile k of a wave's 8, group 4 k + q: lane (row,
// k / 2) holds it at 4 (k % 2) + q of its 8
template <int B>
__device__ __forceinline__ uint32_t code_of(const u32x4& w, int k, int lane)
{
    const int q = lane >> 4, src = ((lane & 15) + 16 * (k >> 1)) * 4;
    if constexpr (B == 2) {
        const uint32_t a = __builtin_amdgcn_ds_bpermute(src, (int)w[2 * (k & 1)]);
        const uint32_t b = __builtin_amdgcn_ds_bpermute(src, (int)w[2 * (k & 1) + 1]);
        return (q & 2 ? b : a) >> (16 * (q & 1)) & 0xFFFFu;
    }
    return (uint32_t)__builtin_amdgcn_ds_bpermute(src, (int)w[k & 1]) >> (8 * q) & 0xFFu;
}

// Forward: rows in plain order.  A wave takes a tile of 16 rows and 8 k
// tiles: lane (row, q) gathers group 4 k + q, and each k tile is one KiB.  The
// codes come 8 a lane where their rows are aligned (vec), and change lanes in
// the LDS unit: loaded one by one they cost a request for each 4 gathers.
// 32768 x 2048 at 2 bits: 50 us, 168 G gathers a second beside 134 MB written.
template <int CBT, int S2, int PARTS>
__global__ void __launch_bounds__(256) dequant_plain_kernel(const DequantArgs a)
{
    constexpr int B1 = S2 == VQ2_S2_U8 ? 1 : 2;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int kt = a.m.ng / 4, k0 = blockIdx.y * 8;
    int mat;
    const int64_t row = mat_row(a.m, a.tile0 + tile, lane & 15, mat);
    const bool ok = row < a.m.rows;
    const int64_t off = (ok ? row : 0) * a.m.ng;
    const void *i0 = a.m.m[mat].i0, *i1 = a.m.m[mat].i1;
    uint32_t c0[8], c1[8];
    if (a.vec) {
        const int g = k0 * 4 + q * 8, at = g < a.m.ng ? g : 0;
        const u32x4 w = codes8<2>(i0, off + at);
        u32x4 v = {0, 0, 0, 0};
        if constexpr (S2 != VQ2_S2_NONE) v = codes8<B1>(i1, off + at);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            c0[k] = code_of<2>(w, k, lane);
            c1[k] = S2 == VQ2_S2_NONE ? 0 : code_of<B1>(v, k, lane);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int64_t i = off + min(k0 + k, kt - 1) * 4 + q;
            c0[k] = ((const uint16_t*)i0)[i];
            c1[k] = code1<S2>(i1, i);
        }
    }
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
    half8_t hi[8], lo[8];
#pragma unroll
    for (int k = 0; k < 8; k++) weight_of<CBT, S2, PARTS>(a.m, c0[k], c1[k], hi[k], lo[k]);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if (k0 + k >= kt) break;
        half8_t* w = a.w + (tile * (PARTS * kt) + k0 + k) * 64 + lane;
        w[0] = ok ? hi[k] : zero;
        if constexpr (PARTS == 2) w[(int64_t)kt * 64] = ok ? lo[k] : zero;
    }
}

// Backward: the rows' panel (WP), and the columns'.  A wave takes 32 rows (two
// tiles) and 16 groups: lane (q, g) gathers the 8 rows of chunk q of group g.
// Column j of the 8 centroids is then one operand of the columns' panel, whose
// block j holds columns j, 8 + j, ... of the 16 groups: one KiB a block, and a
// lane of the next product holds 8 neighbouring columns in its 8 row tiles.
// 16384 x 2048 at 2 bits: 40 us, 105 G gathers a second beside 134 MB written (27 us at
// a large copy's rate); the conflicts of its LDS writes (82 % of its LDS cycles) cost
// nothing, 40 us without them, too.
template <int CBT, int S2, int WP, int TP>
__global__ void __launch_bounds__(256) dequant_both_kernel(const DequantArgs a)
{
    const int lane = threadIdx.x & 63, c = lane >> 4, g = blockIdx.y * 16 + (lane & 15);
    const int pair = blockIdx.x * 4 + (threadIdx.x >> 6);  // of the piece
    const int kt = a.m.ng / 4;
    const bool g_ok = g < a.m.ng;
    uint32_t c0[8], c1[8];
    bool ok[8];
#pragma unroll
    for (int m = 0; m < 8; m++) {
        int mat;
        const int64_t row = mat_row(a.m, a.tile0 + 2 * pair + m / 4, 4 * c + m % 4, mat);
        ok[m] = g_ok && row < a.m.rows;
        const int64_t i = ok[m] ? row * a.m.ng + g : 0;
        c0[m] = ((const uint16_t*)a.m.m[mat].i0)[i];
        c1[m] = code1<S2>(a.m.m[mat].i1, i);
    }
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
    constexpr int PARTS = WP == 2 || TP == 2 ? 2 : 1;
    half8_t hi[8], lo[8];
#pragma unroll
    for (int m = 0; m < 8; m++) weight_of<CBT, S2, PARTS>(a.m, c0[m], c1[m], hi[m], lo[m]);
#pragma unroll
    for (int m = 0; m < 8; m++) {
        hi[m] = ok[m] ? hi[m] : zero;
        if constexpr (PARTS == 2) lo[m] = ok[m] ? lo[m] : zero;
    }
    if constexpr (WP != 0) {
        // the wave's 2 row tiles by 4 k tiles, a KiB each, put in order in LDS
        __shared__ half8_t s_w[4][8][64];
        half8_t(*sw)[64] = s_w[threadIdx.x >> 6];
        const int gi = lane & 15, k0 = blockIdx.y * 4;
#pragma unroll
        for (int part = 0; part < WP; part++) {
#pragma unroll
            for (int m = 0; m < 8; m++) sw[(m / 4) * 4 + gi / 4][(gi & 3) * 16 + 4 * c + m % 4] = part ? lo[m] : hi[m];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int f = 0; f < 8; f++)
                if (k0 + f % 4 < kt) a.w[((int64_t)(2 * pair + f / 4) * (WP * kt) + part * kt + k0 + f % 4) * 64 + lane] = sw[f][lane];
            __builtin_amdgcn_wave_barrier();
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        half8_t* t = a.wt + ((int64_t)(blockIdx.y * 8 + j) * (TP * a.vkt) + pair) * 64 + lane;
        half8_t v;
#pragma unroll
        for (int m = 0; m < 8; m++) v[m] = hi[m][j];
        t[0] = v;
        if constexpr (TP == 2) {
#pragma unroll
            for (int m = 0; m < 8; m++) v[m] = lo[m][j];
            t[(int64_t)a.vkt * 64] = v;
        }
    }
}

// -------------------------------------------------------------- epilogues
// What a product of weights (panel a) and tokens (panel b) is made into.
// `tile` is the first weight tile of the wave, counted over all pieces, `tok`
// its first token.

constexpr int64_t TARGET_SKIP = -1, TARGET_BAD = -2;
// the token's target, TARGET_SKIP for a token that does not count, TARGET_BAD
// for one outside the vocabulary
__device__ __forceinline__ int64_t target_of(const int64_t* t, int64_t i, int64_t ignore, int64_t rows)
{
    const int64_t v = t[i];
    return v == ignore ? TARGET_SKIP : v < 0 || v >= rows ? TARGET_BAD : v;
}

// row scale * rs of row r of matrix `mat`; 0 past the last row
__device__ __forceinline__ float row_scale(const MatArgs& m, float rs, int mat, int64_t r)
{
    return r < m.rows ? load_as_f32(m.m[mat].scale, m.s_dt, r) * rs : 0.0f;
}

struct StatsEpi {
    const float* sc;
    const float* fac;
    const int64_t* target;
    int64_t rows, ignore;
    int tokens, tp;
    f32x2_t* part;  // [parts of rows][tp]: largest logit and sum of exp(l - largest)
    float* at;      // [tp]: the target's logit
    // few_kernel: a lane's running maximum and sum for its token
    struct State {
        float m = NEG_INF, s = 0.0f;
    };
    __device__ __forceinline__ void few(State& st, const MatArgs& m, float rs, f32x4_t a, f32x4_t b, int64_t pair, int t) const
    {
        const int q = (threadIdx.x & 63) >> 4;
        const int64_t r0 = pair * 32 + q * 4;
        float z[8], top = st.m;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int64_t r = r0 + (k >> 2) * 16 + (k & 3);
            z[k] = r < m.rows ? (k < 4 ? a[k & 3] : b[k & 3]) * row_scale(m, rs, 0, r) : NEG_INF;
            top = fmaxf(top, z[k]);
        }
        const float base = top == NEG_INF ? 0.0f : top;
        st.s *= __expf(st.m - base);
        st.m = top;
#pragma unroll
        for (int k = 0; k < 8; k++) st.s += __expf(z[k] - base);
        const int64_t rel = (t < tokens ? target_of(target, t, ignore, rows) : TARGET_SKIP) - r0;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (rel == (k >> 2) * 16 + (k & 3)) at[t] = z[k];
    }
    __device__ __forceinline__ void few_end(const State& st, int64_t chunk, int t) const
    {
        const float top = max_rows(st.m), base = top == NEG_INF ? 0.0f : top;
        const float sum = sum_rows(st.s * __expf(st.m - base));
        if ((threadIdx.x & 63) < 16) part[chunk * tp + t] = f32x2_t{top, sum};
    }
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
        f32x4_t s[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) s[i] = *(const f32x4_t*)(sc + (tile + i) * 16 + q * 4);
        const bool tail = (tile + MT) * 16 > rows;
#pragma unroll
        for (int j = 0; j < PG_NT; j++) {
            const int t = tok + j * 16 + nl;
            const float f = fac[t];
            float m = NEG_INF;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float z = acc[i][j][e] * f * s[i][e];
                    if (tail && (tile + i) * 16 + q * 4 + e >= rows) z = NEG_INF;
                    acc[i][j][e] = z;
                    m = fmaxf(m, z);
                }
            m = max_rows(m);
            const float base = m == NEG_INF ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum += __expf(acc[i][j][e] - base);
            sum = sum_rows(sum);
            if (q == 0) part[(tile / MT) * tp + t] = f32x2_t{m, sum};
            const int64_t v = t < tokens ? target_of(target, t, ignore, rows) : TARGET_SKIP;
            const int64_t rel = v - tile * 16;
            if (rel >= 0 && rel < MT * 16) {  // (few lanes of a launch)
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (rel == i * 16 + q * 4 + e) at[t] = acc[i][j][e];
            }
        }
    }
};

struct DlogitEpi {
    const float* sc;
    const float* fac;
    const float* lse;
    const float* dloss;
    const int64_t* target;
    RowTop amax;
    int64_t rows, ignore, tile0;  // tile0: the piece's first tile
    int tokens, tp, vkt;
    half8_t* p;    // the next product's panel of tokens, [tp / 16][vkt][64]
    float* ds;     // [tp / 64][16 * all tiles]: sums over 64 tokens, or null
    int64_t ds_ld;
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
        const float c = pow2(14 - scale_exponent(amax));
        // A token that does not count has a row of zeros and an infinite l: no term
        // of it is anything but 0.
        float l[PG_NT], upf[PG_NT], f[PG_NT];
        int rel[PG_NT];   // the target's row of the wave's, or none
        bool hit[PG_NT];  // some lane's
#pragma unroll
        for (int j = 0; j < PG_NT; j++) {
            const int t = tok + j * 16 + nl;
            int64_t v = TARGET_SKIP;
            l[j] = __builtin_inff();
            upf[j] = 0.0f;
            f[j] = fac[t];
            if (t < tokens) v = target_of(target, t, ignore, rows);
            if (v != TARGET_SKIP) {
                l[j] = lse[t];
                upf[j] = v == TARGET_BAD ? __builtin_nanf("") : dloss[t] * f[j];
            }
            const int64_t r = v - tile * 16;
            rel[j] = r >= 0 && r < MT * 16 ? (int)r : -1;
            hit[j] = __any(rel[j] >= 0);
        }
        const int left = (int)min(rows - tile * 16, (int64_t)MT * 16);  // rows of the wave that exist
        const bool tail = left < MT * 16;
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
            f32x4_t s[2], d[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                s[k] = *(const f32x4_t*)(sc + (tile + i + k) * 16 + q * 4);
                d[k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int j = 0; j < PG_NT; j++) {
                float v[8];
#pragma unroll
                for (int m = 0; m < 8; m++) v[m] = __expf(acc[i + (m >> 2)][j][m & 3] * f[j] * s[m >> 2][m & 3] - l[j]);
                if (hit[j]) {  // (few waves)
#pragma unroll
                    for (int m = 0; m < 8; m++) v[m] -= rel[j] == (i + (m >> 2)) * 16 + 4 * q + (m & 3) ? 1.0f : 0.0f;
                }
                if (tail) {
#pragma unroll
                    for (int m = 0; m < 8; m++)
                        if ((i + (m >> 2)) * 16 + 4 * q + (m & 3) >= left) v[m] = 0.0f;
                }
                half8_t h;
#pragma unroll
                for (int m = 0; m < 8; m++) {
                    const int e = m & 3, k = m >> 2;
                    h[m] = (_Float16)(v[m] * (s[k][e] * c));
                    if (ds) d[k][e] += v[m] * (acc[i + k][j][e] * upf[j]);
                }
                p[((int64_t)((tok >> 4) + j) * vkt + (tile - tile0 + i) / 2) * 64 + lane] = h;
            }
            if (ds) {
#pragma unroll
                for (int m = 0; m < 8; m++) {
                    const float v = group_sum(d[m >> 2][m & 3], 16);
                    if (nl == 0) ds[(tok / (16 * PG_NT)) * ds_ld + (tile + i + (m >> 2)) * 16 + q * 4 + (m & 3)] = v;
                }
            }
        }
    }
};

// f(g), and its derivative
template <int ACT>
__device__ __forceinline__ void gate_act(float g, float& f, float& df)
{
    if constexpr (ACT == VQ2_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));  // (2^-23 of it; a division's 10 instructions show)
        f = g * s;
        df = s * (1.0f + g * (1.0f - s));
        if (g == NEG_INF) f = df = 0.0f;  // (below -87 the sigmoid is no normal number: 0)
    } else {
        // g / (1 + exp(-2 u)), u the tanh form's argument
        const float g2 = g * g, u2 = 1.5957691216057308f * g * (1.0f + 0.044715f * g2);
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-u2));
        f = g * s;
        df = s * (1.0f + g * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * g2)));
        if (g < -12.0f) f = df = 0.0f;
        if (g > 12.0f) { f = g; df = 1.0f; }
    }
}

struct GatedEpi {
    const float* sc;
    const float* fac;
    void* y;
    int y_dt, tokens;
    int64_t rows;
    int vec;  // rows a multiple of 4, y aligned: 4 values a store
    int act;
    __device__ __forceinline__ void store(int t, int64_t r0, const float (&o)[4]) const
    {
        const int64_t at = (int64_t)t * rows + r0;
        if (!vec) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (r0 + e < rows) store_from_f32(y, y_dt, at + e, o[e]);
        } else if (y_dt == VQ2_DT_F32) {
            *(f32x4_t*)((float*)y + at) = f32x4_t{o[0], o[1], o[2], o[3]};
        } else if (y_dt == VQ2_DT_F16) {
            *(half4_t*)((uint16_t*)y + at) = half4_t{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
        } else {
            *(u32x2*)((uint16_t*)y + at) = u32x2{bf16_pair(o[0], o[1]), bf16_pair(o[2], o[3])};
        }
    }
    struct State {};
    __device__ __forceinline__ void few_end(const State&, int64_t, int) const {}
    __device__ __forceinline__ void few(State&, const MatArgs& m, float rs, f32x4_t g, f32x4_t u, int64_t pair, int t) const
    {
        const int q = (threadIdx.x & 63) >> 4;
        const int64_t r0 = pair * 16 + q * 4;
        if (t >= tokens || r0 >= rows) return;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float v = g[e] * row_scale(m, rs, 0, r0 + e);
            float f, df;
            if (act == VQ2_ACT_SILU) gate_act<VQ2_ACT_SILU>(v, f, df);
            else gate_act<VQ2_ACT_GELU_TANH>(v, f, df);
            o[e] = f * (u[e] * row_scale(m, rs, 1, r0 + e));
        }
        store(t, r0, o);
    }
    template <int ACT, int MT>
    __device__ __forceinline__ void run_act(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
            const f32x4_t sg = *(const f32x4_t*)(sc + (tile + i) * 16 + q * 4);
            const f32x4_t su = *(const f32x4_t*)(sc + (tile + i + 1) * 16 + q * 4);
            const int64_t r0 = (tile + i) / 2 * 16 + q * 4;
#pragma unroll
            for (int j = 0; j < PG_NT; j++) {
                const int t = tok + j * 16 + nl;
                if (t >= tokens || r0 >= rows) continue;
                const float x = fac[t];
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float f, df;
                    gate_act<ACT>(acc[i][j][e] * x * sg[e], f, df);
                    o[e] = f * (acc[i + 1][j][e] * x * su[e]);
                }
                store(t, r0, o);
            }
        }
    }
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int)
    {
        if (act == VQ2_ACT_SILU) run_act<VQ2_ACT_SILU>(acc, tile, tok);
        else run_act<VQ2_ACT_GELU_TANH>(acc, tile, tok);
    }
};

// Upstream values of 4 neighbouring rows of a token, as loaded and as numbers.
// V16: 16-bit rows by 8 bytes; otherwise fp32 rows by 16 (vec), or one by one (all
// three in one kernel: the block's step of 4096 tokens 670.6 -> 673.2 us).
struct UpstreamArgs {
    const void* dy;  // [tokens][rows]
    int dt, tokens, vec;
    int64_t rows;
};
template <bool V16>
struct Upstream : UpstreamArgs {
    // (past the tokens or rows: anything of the row, which is dropped)
    __device__ __forceinline__ int64_t place(int t, int64_t r) const
    {
        return (int64_t)min(t, tokens - 1) * rows + (r < rows ? r : 0);
    }
    __device__ __forceinline__ u32x2 raw(int t, int64_t r) const { return *(const u32x2*)((const uint16_t*)dy + place(t, r)); }
    __device__ __forceinline__ f32x4_t words(int t, int64_t r) const { return *(const f32x4_t*)((const float*)dy + place(t, r)); }
    __device__ __forceinline__ f32x4_t kept(f32x4_t v, int t, int64_t r) const
    {
        const bool in = t < tokens && r < rows;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = in ? v[e] : 0.0f;
        return v;
    }
    __device__ __forceinline__ f32x4_t numbers(u32x2 w, int t, int64_t r) const
    {
        f32x4_t v;
        if (dt == VQ2_DT_F16) {
            const half4_t h = __builtin_bit_cast(half4_t, w);
            v = f32x4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        } else {
            v = f32x4_t{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                        __uint_as_float(w.y & 0xFFFF0000u)};
        }
        return kept(v, t, r);
    }
    __device__ __forceinline__ f32x4_t slow(int t, int64_t r) const
    {
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (t < tokens && r + e < rows) v[e] = load_as_f32(dy, dt, (int64_t)t * rows + r + e);
        return v;
    }
    // of PG_NT token tiles
    __device__ __forceinline__ void load(f32x4_t (&d)[PG_NT], int t, int64_t r) const
    {
        if constexpr (V16) {
            u32x2 w[PG_NT];
#pragma unroll
            for (int j = 0; j < PG_NT; j++) w[j] = raw(t + j * 16, r);
#pragma unroll
            for (int j = 0; j < PG_NT; j++) d[j] = numbers(w[j], t + j * 16, r);
        } else if (vec) {
#pragma unroll
            for (int j = 0; j < PG_NT; j++) d[j] = words(t + j * 16, r);
#pragma unroll
            for (int j = 0; j < PG_NT; j++) d[j] = kept(d[j], t + j * 16, r);
        } else {
#pragma unroll
            for (int j = 0; j < PG_NT; j++) d[j] = slow(t + j * 16, r);
        }
    }
};

template <bool V16>
struct DgatedEpi {
    const float* sc;
    const float* fac;
    const float* dfac;  // [tp]: 2^-e of the token's upstream row (dy_max)
    Upstream<V16> up;
    BlockBound bound;
    int tp, vkt;
    int64_t tile0;
    half8_t* p;
    float* ds;
    int64_t ds_ld;
    int act;
    template <int ACT, int MT>
    __device__ __forceinline__ void run_act(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
        const float c = pow2(-scale_exponent(bound.amax));
        const int common = bound.common();
        float x[PG_NT], k[PG_NT], b[PG_NT];  // (two factors: their product may leave fp32's range)
#pragma unroll
        for (int j = 0; j < PG_NT; j++) {
            x[j] = fac[tok + j * 16 + nl];
            k[j] = dfac[tok + j * 16 + nl];
            b[j] = pow2_near(-bound.of(common, tok + j * 16 + nl));
        }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
            const f32x4_t sg = *(const f32x4_t*)(sc + (tile + i) * 16 + q * 4);
            const f32x4_t su = *(const f32x4_t*)(sc + (tile + i + 1) * 16 + q * 4);
            f32x4_t d[PG_NT];
            up.load(d, tok + nl, (tile + i) / 2 * 16 + q * 4);
            f32x4_t dsg = {0.0f, 0.0f, 0.0f, 0.0f}, dsu = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < PG_NT; j++) {
                half8_t h;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float rg = acc[i][j][e] * x[j], ru = acc[i + 1][j][e] * x[j];
                    float f, df;
                    gate_act<ACT>(rg * sg[e], f, df);
                    const float dg = d[j][e] * (ru * su[e]) * df, du = d[j][e] * f;
                    h[e] = (_Float16)(dg * k[j] * b[j] * (sg[e] * c));
                    h[4 + e] = (_Float16)(du * k[j] * b[j] * (su[e] * c));
                    if (ds) {
                        dsg[e] += dg * rg;
                        dsu[e] += du * ru;
                    }
                }
                p[((int64_t)((tok >> 4) + j) * vkt + (tile - tile0 + i) / 2) * 64 + lane] = h;
            }
            if (ds) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = group_sum(dsg[e], 16), b = group_sum(dsu[e], 16);
                    if (nl == 0) {
                        float* o = ds + (tok / (16 * PG_NT)) * ds_ld + (tile + i) * 16 + q * 4 + e;
                        o[0] = a;
                        o[16] = b;
                    }
                }
            }
        }
    }
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int)
    {
        if (act == VQ2_ACT_SILU) run_act<VQ2_ACT_SILU>(acc, tile, tok);
        else run_act<VQ2_ACT_GELU_TANH>(acc, tile, tok);
    }
};

// sums over 64 tokens of upstream times product: the row scales' gradient
template <bool V16>
struct ColsumEpi {
    const float* fac;
    Upstream<V16> up;
    float* ds;
    int64_t ds_ld;
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
        float x[PG_NT];
#pragma unroll
        for (int j = 0; j < PG_NT; j++) x[j] = fac[tok + j * 16 + nl];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            f32x4_t u[PG_NT], d = {0.0f, 0.0f, 0.0f, 0.0f};
            up.load(u, tok + nl, (tile + i) * 16 + q * 4);
#pragma unroll
            for (int j = 0; j < PG_NT; j++) d += u[j] * (acc[i][j] * x[j]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = group_sum(d[e], 16);
                if (nl == 0) ds[(tok / (16 * PG_NT)) * ds_ld + (tile + i) * 16 + q * 4 + e] = v;
            }
        }
    }
};

// What makes a row of the columns' product one of dx: the factors that its
// panel left out, and of the loss the upstream value (zero rows: exactly zero).
struct DxFactor {
    RowTop amax;
    const float* dfac;  // [tp], or null: the loss's
    const float* dloss;
    const int64_t* target;
    int64_t rows, ignore;
    BlockBound bound;   // of the block; bits 0: none
    int e;              // by init(), called by whole waves
    // (two factors: their product may leave fp32's range)
    struct Of {
        float a, b;
        bool skip;
        __device__ __forceinline__ float operator()(float v) const { return skip ? 0.0f : v * b * a; }
    };
    __device__ __forceinline__ void init()
    {
        e = scale_exponent(amax) - (dfac ? 0 : 14);
        if (bound.bits) e += bound.common();
    }
    __device__ __forceinline__ Of of(int t) const
    {
        if (dfac) return Of{1.0f / dfac[t], pow2_near(bound.bits ? bound.of(e, t) : e), false};
        const int64_t v = target_of(target, t, ignore, rows);
        return Of{v == TARGET_BAD ? __builtin_nanf("") : dloss[t], pow2(e), v == TARGET_SKIP};
    }
};

// 8 (4) neighbouring columns of dx: element e of N tiles' values
template <int N>
__device__ __forceinline__ void store_run(void* dx, int dt, int64_t at, const f32x4_t (&v)[N], int e, const DxFactor::Of& f)
{
    if (dt == VQ2_DT_F32) {
        f32x4_t* o = (f32x4_t*)((float*)dx + at);
#pragma unroll
        for (int i = 0; i < N; i += 4) o[i / 4] = f32x4_t{f(v[i][e]), f(v[i + 1][e]), f(v[i + 2][e]), f(v[i + 3][e])};
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float a = f(v[i][e]), b = f(v[i + 1][e]);
        w[i / 2] = dt == VQ2_DT_F16 ? f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16 : bf16_pair(a, b);
    }
    uint32_t* o = (uint32_t*)((uint16_t*)dx + at);
    if constexpr (N == 8) *(u32x4*)o = u32x4{w[0], w[1], w[2], w[3]};
    else *(u32x2*)o = u32x2{w[0], w[1]};
}

// Columns' product, added to what earlier pieces left, or (dx) finished: tile i
// of the wave holds columns i, 8 + i, ... of its 128 (MT == 8), or of the half
// of them that starts at tile % 8.
struct GradEpi {
    f32x4_t* out;  // as the lanes hold them: [slices][tp / 16][np / 128][8][64] (dx_kernel)
    int64_t np;
    int tp, add;
    void* dx;    // [tokens][n], or null
    int dx_dt, tokens, n;
    DxFactor fac;
    template <int MT>
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][PG_NT], int64_t tile, int tok, int bz)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4, nl = lane & 15;
        const int64_t c0 = tile / 8 * 128 + tile % 8;
        if (dx) {
            fac.init();
#pragma unroll
            for (int j = 0; j < PG_NT; j++) {
                const int t = tok + j * 16 + nl;
                if (t >= tokens) continue;
                const DxFactor::Of f = fac.of(t);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t col = c0 + (q * 4 + e) * 8;
                    if (col >= n) continue;
                    f32x4_t v[MT];
#pragma unroll
                    for (int i = 0; i < MT; i++) v[i] = acc[i][j];
                    store_run(dx, dx_dt, (int64_t)t * n + col, v, e, f);
                }
            }
            return;
        }
        // (in rows, 16 bytes a lane and line, the loss's 4096 x 2048 sums cost 25
        // us a piece more)
#pragma unroll
        for (int j = 0; j < PG_NT; j++) {
            f32x4_t* o = out + ((((int64_t)bz * (tp / 16) + (tok >> 4) + j) * (np / 128) + tile / 8) * 8 + tile % 8) * 64 + lane;
#pragma unroll
            for (int i = 0; i < MT; i++) o[i * 64] = add ? o[i * 64] + acc[i][j] : acc[i][j];
        }
    }
};

template <int MT, class Epi>
__global__ void __launch_bounds__(PG_THREADS, MT == 8 ? 2 : 3) panel_gemm_kernel(const PanelGemmArgs g, Epi epi, int64_t tile0)
{
    int bm, bn, bz;
    panel_tile(g, bm, bn, bz);
    f32x4_t acc[MT][PG_NT];
    panel_product<MT>(g, bm, bn, bz, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % PG_WM, wn = wave / PG_WM;
    epi.template run<MT>(acc, tile0 + (bm * PG_WM + wm) * MT, (bn * PG_WN + wn) * PG_NT * 16, bz);
}

// ------------------------------------------------------------ upstream rows
template <bool V16>
struct DyArgs {
    Upstream<V16> up;
    int64_t row0;     // the piece's first
    const float* sc;
    RowTop amax;
    const float* dfac;
    half8_t* p;       // [tp / 16][vkt][64]
    int vkt;
};
// The panel of dy * scale * 2^-e in the order of the columns' panel:
// two runs of 4 rows a lane.  A wave 4 k tiles of 16 tokens.
template <bool V16>
__global__ void __launch_bounds__(256) dy_panel_kernel(const DyArgs<V16> a)
{
    constexpr int N = 4;
    const int lane = threadIdx.x & 63, q = lane >> 4, tile = blockIdx.x, t = tile * 16 + (lane & 15);
    const int k0 = ((int)blockIdx.y * 4 + (threadIdx.x >> 6)) * N;
    // (two factors: their product may leave fp32's range)
    const float f = a.dfac[t], c = pow2(-scale_exponent(a.amax));
    f32x4_t v[N][2], s[N][2];
    if constexpr (V16) {
        u32x2 w[N][2];
#pragma unroll
        for (int i = 0; i < 2 * N; i++) w[i / 2][i % 2] = a.up.raw(t, a.row0 + (k0 + i / 2) * 32 + i % 2 * 16 + q * 4);
#pragma unroll
        for (int i = 0; i < 2 * N; i++)
            v[i / 2][i % 2] = a.up.numbers(w[i / 2][i % 2], t, a.row0 + (k0 + i / 2) * 32 + i % 2 * 16 + q * 4);
    } else if (a.up.vec) {
#pragma unroll
        for (int i = 0; i < 2 * N; i++) v[i / 2][i % 2] = a.up.words(t, a.row0 + (k0 + i / 2) * 32 + i % 2 * 16 + q * 4);
#pragma unroll
        for (int i = 0; i < 2 * N; i++)
            v[i / 2][i % 2] = a.up.kept(v[i / 2][i % 2], t, a.row0 + (k0 + i / 2) * 32 + i % 2 * 16 + q * 4);
    } else {
#pragma unroll
        for (int i = 0; i < 2 * N; i++) v[i / 2][i % 2] = a.up.slow(t, a.row0 + (k0 + i / 2) * 32 + i % 2 * 16 + q * 4);
    }
#pragma unroll
    for (int i = 0; i < 2 * N; i++) s[i / 2][i % 2] = *(const f32x4_t*)(a.sc + a.row0 + min(k0 + i / 2, a.vkt - 1) * 32 + i % 2 * 16 + q * 4);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (k0 + i >= a.vkt) break;
        half8_t h;
#pragma unroll
        for (int m = 0; m < 8; m++) h[m] = (_Float16)(v[i][m >> 2][m & 3] * f * (s[i][m >> 2][m & 3] * c));
        a.p[((int64_t)tile * a.vkt + k0 + i) * 64 + lane] = h;
    }
}

// ------------------------------------------------------------- few tokens
// Every centroid is gathered once for up to 128 tokens, straight into the
// operand it is (lane (row, q): group q of a k tile), and nothing is written in
// between.  The gathers bound it: 240 G a second over the device, whatever
// their size (a request of a line each): one token of a 151936 x 2048 head (38.9 M
// codes, 162 us by them) takes 171 us, of the block of 2 x 6144 x 2048 at 4 bits (6.3 M,
// 26 us) 34.  A wave takes two tiles of 16 rows (for the block: gate and up).
// The 4 waves of a workgroup share the k tiles of one pair and meet in LDS, so
// that small matrices fill the device; with many rows and more than 64 tokens
// each has a pair of its own (few_alone), and they share the tokens' lines.
//
// k tiles in groups of 8: lane q takes the groups 8 q + j (j = tile of the 8)
// of 32, so its 8 codes are one load (from any address: vector loads take
// those), and the tokens' operand is read from there, too.  Up to 4 tokens are read as they are (no launch before): a wave
// brings its share of a token's row to fp16 under a power of two of its own.
typedef uint32_t codes16_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t codes8_t __attribute__((ext_vector_type(2), aligned(1)));
struct FewArgs {
    MatArgs m;
    int64_t pairs;
    const half8_t* xp;  // packed tokens
    const float* fac;
    const void* x;      // OWN: 16-bit rows as they are
    int x_dt;
    int tokens, n;  // tokens of the chunk; workgroups (., y) take 16 TT of them from 16 TT y on
    float rs;
};

// a gathered centroid in fp16
template <int CBT>
__device__ __forceinline__ half8_t centroid_f16(half8_t h)
{
    if constexpr (CBT == VQ2_DT_BF16) {
        const u32x4 u = __builtin_bit_cast(u32x4, h);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            h[2 * k] = (_Float16)__uint_as_float(u[k] << 16);
            h[2 * k + 1] = (_Float16)__uint_as_float(u[k] & 0xFFFF0000u);
        }
    }
    return h;
}

template <int CBT, int S2, int TT, int KW, bool OWN, class Epi>
__global__ void __launch_bounds__(256, TT >= 6 || OWN ? 2 : 3) few_kernel(const FewArgs a, Epi epi)
{
    static_assert((KW == 4 || KW == 1) && (!OWN || (TT == 1 && KW == 4)), "");
    constexpr int JU = S2 == VQ2_S2_NONE && TT <= 4 ? 8 : 4;  // k tiles whose centroids are on their way together
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, nl = lane & 15;
    const int tok0 = blockIdx.y * (16 * TT), left = a.tokens - tok0;
    const int ng = a.m.ng, kt = ng / 4, sups = (ng + 31) / 32, part = KW == 4 ? wave : 0;
    const int s0 = sups * part / KW, s1 = sups * (part + 1) / KW;
    const half8_t* xp = a.xp + (int64_t)(tok0 / 16) * kt * 64;
    const int64_t step = (int64_t)gridDim.x * (4 / KW);
    int64_t pair = KW == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    const int16_t* p0[2];
    const char* p1[2];
    constexpr int B1 = S2 == VQ2_S2_U8 ? 1 : 2;
    auto set_pair = [&] {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int mat;
            const int64_t row = mat_row(a.m, 2 * min(pair, a.pairs - 1) + i, nl, mat), off = (row < a.m.rows ? row : 0) * ng;
            p0[i] = a.m.m[mat].i0 + off;
            p1[i] = S2 == VQ2_S2_NONE ? nullptr : (const char*)a.m.m[mat].i1 + off * B1;
        }
    };
    set_pair();
    struct Codes {
        u32x4 a[2], b[S2 == VQ2_S2_NONE ? 1 : 2];
    };
    auto load_codes = [&](int sup, Codes& c) {
        const int g = min(sup, sups - 1) * 32 + q * 8, at = g < ng ? g : 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            c.a[i] = *(const codes16_t*)(p0[i] + at);
            if constexpr (S2 == VQ2_S2_U16) c.b[i] = *(const codes16_t*)(p1[i] + at * 2);
            if constexpr (S2 == VQ2_S2_U8) {
                const u32x2 u = *(const codes8_t*)(p1[i] + at);
                c.b[i].x = u.x;
                c.b[i].y = u.y;
            }
        }
    };
    auto code = [](const u32x4& w, int j) { return w[j >> 1] >> (16 * (j & 1)) & 0xFFFFu; };
    Codes cur, next;
    load_codes(min(s0, sups - 1), cur);

    // the tokens of a wave that reads them itself: their largest values first
    float up = 1.0f, down = 1.0f;  // 2^e, 2^-e of token nl
    auto raw_x = [&](int s, u32x4 (&w)[8]) {  // 16-bit values of token nl, the lane's 8 groups
        const int g = s * 32 + q * 8 < ng ? s * 32 + q * 8 : 0;
        const u32x4* p = (const u32x4*)((const uint16_t*)a.x + (int64_t)min(nl, a.tokens - 1) * a.n + g * 8);
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = p[j];
    };
    auto eight = [&](const u32x4& w) {
        Eight e;
        if (a.x_dt == VQ2_DT_F16) {
            const half8_t h = __builtin_bit_cast(half8_t, w);
#pragma unroll
            for (int k = 0; k < 8; k++) e.v[k] = (float)h[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                e.v[2 * k] = __uint_as_float(w[k] << 16);
                e.v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
            }
        }
        return e;
    };
    u32x4 xw[OWN ? 8 : 1];
    if constexpr (OWN) {
        float m = 0.0f;
        for (int s = s1 - 1; s >= s0; s--) {  // the first last: it is used first
            raw_x(s, xw);
            if (s * 32 + q * 8 < ng)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const Eight e = eight(xw[j]);
#pragma unroll
                    for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(e.v[k]));
                }
        }
        m = max_rows(m);
        const int e = m > 0.0f ? min(max(exponent_of(m) - 13, -110), 110) : 0;
        up = pow2(e);
        down = pow2(-e);
    }

    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
    constexpr int TS = KW == 4 ? (TT + 3) / 4 : TT;  // token tiles that this wave finishes: wave, wave + 4, ...
    typename Epi::State state[TS];
    // The tokens' operand of the next k tile is on its way while one is multiplied,
    // where a wave is often alone on its SIMD (333 tokens of 2 x 1000 x 2048: 26.9 us
    // without, 25.0; 3 ahead 29.5).  With rows of its own, or two stages' centroids beside
    // it, it would take registers that loads in flight need (96 tokens of 50257 rows
    // 99.1 -> 100.5, 64 of 2 x 1000 at 3 bits 19.9 -> 21.1).
    constexpr int R = OWN || KW == 1 || S2 != VQ2_S2_NONE ? 1 : 2;
    half8_t b[R][TT];
    auto load_b = [&](int s, int j, half8_t (&o)[TT]) {
        const int g = s * 32 + q * 8 < ng ? s * 32 + q * 8 + j : 0;
#pragma unroll
        for (int t = 0; t < TT; t++) o[t] = xp[((int64_t)t * kt + (g >> 2)) * 64 + (g & 3) * 16 + nl];
    };
    if constexpr (!OWN)
#pragma unroll
        for (int j = 0; j < R - 1; j++) load_b(s0, j, b[j]);
    for (; pair < a.pairs;) {
    f32x4_t acc[2][TT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = s0; s < s1; s++) {
        const bool ok = s * 32 + q * 8 < ng;
        if constexpr (OWN)
            if (s1 - s0 > 1) raw_x(s, xw);
        if (s + 1 == s1) {  // the next pair's first codes
            pair += step;
            set_pair();
        }
        load_codes(s + 1 == s1 ? s0 : s + 1, next);
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += JU) {
            half8_t w0[2][JU], w1[2][S2 == VQ2_S2_NONE ? 1 : JU];
#pragma unroll
            for (int u = 0; u < JU; u++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int j = j0 + u;
                    w0[i][u] = ((const half8_t*)a.m.cb0)[code(cur.a[i], j)];
                    if constexpr (S2 == VQ2_S2_U16) w1[i][u] = ((const half8_t*)a.m.cb1)[code(cur.b[i], j)];
                    if constexpr (S2 == VQ2_S2_U8) w1[i][u] = ((const half8_t*)a.m.cb1)[cur.b[i][j >> 2] >> (8 * (j & 3)) & 0xFFu];
                }
#pragma unroll
            for (int u = 0; u < JU; u++) {
                const int j = j0 + u, at = j % R;
                if constexpr (OWN) {
                    const Eight e = eight(xw[j]);
#pragma unroll
                    for (int k = 0; k < 8; k++) b[at][0][k] = (_Float16)(e.v[k] * down);
                } else {
                    load_b(j + R - 1 < 8 ? s : s + 1 == s1 ? s0 : s + 1, (j + R - 1) % 8, b[(j + R - 1) % R]);
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const half8_t w = ok ? centroid_f16<CBT>(w0[i][u]) : zero;
#pragma unroll
                    for (int t = 0; t < TT; t++) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, b[at][t], acc[i][t], 0, 0, 0);
                    if constexpr (S2 != VQ2_S2_NONE) {
                        const half8_t v = ok ? centroid_f16<CBT>(w1[i][u]) : zero;
#pragma unroll
                        for (int t = 0; t < TT; t++)
                            acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, b[at][t], acc[i][t], 0, 0, 0);
                    }
                }
            }
        }
        cur = next;
    }
    const int64_t done = s1 > s0 ? pair - step : pair;
    if constexpr (KW == 4) {
        if (s1 <= s0) pair += step;  // (a wave without k tiles: rows below 128 values)
        __shared__ f32x4_t s_acc[4][TT][64];
        f32x4_t o[TS][2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            __syncthreads();  // what was there has been read
#pragma unroll
            for (int t = 0; t < TT; t++) s_acc[wave][t][lane] = acc[i][t] * up;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < TS; k++) {
                const int t = min(wave + 4 * k, TT - 1);
                o[k][i] = s_acc[0][t][lane];
#pragma unroll
                for (int w = 1; w < 4; w++) o[k][i] += s_acc[w][t][lane];
            }
        }
#pragma unroll
        for (int k = 0; k < TS; k++) {
            const int t = wave + 4 * k;
            if (t >= TT || t * 16 >= left) break;
            const int tok = tok0 + t * 16 + nl;
            const float f = OWN ? 1.0f : a.fac[tok];
            epi.few(state[k], a.m, a.rs, o[k][0] * f, o[k][1] * f, done, tok);
        }
    } else {
#pragma unroll
        for (int t = 0; t < TT; t++) {
            if (t * 16 >= left) break;
            const int tok = tok0 + t * 16 + nl;
            const float f = a.fac[tok];
            epi.few(state[t], a.m, a.rs, acc[0][t] * f, acc[1][t] * f, done, tok);
        }
    }
    }
#pragma unroll
    for (int k = 0; k < TS; k++) {
        const int t = KW == 4 ? wave + 4 * k : k;
        if (t < TT && t * 16 < left) epi.few_end(state[k], KW == 4 ? blockIdx.x : blockIdx.x * 4 + wave, tok0 + t * 16 + nl);
    }
}

// ---------------------------------------------------------------- last steps
struct LseArgs {
    const f32x2_t* part;
    int64_t chunks;
    int tokens, tp;
    const int64_t* target;
    int64_t rows, ignore;
    const float* at;
    float* loss;
    float* lse;
};
// 16 tokens a workgroup, 64 threads a token over the chunks
constexpr int LSE_LANES = 64;
__global__ void __launch_bounds__(16 * LSE_LANES) lse_kernel(const LseArgs a)
{
    __shared__ f32x2_t s_p[LSE_LANES][17];
    const int tid = threadIdx.x, tl = tid & 15, t = blockIdx.x * 16 + tl;
    float m = NEG_INF, s = 0.0f;
    auto add = [&](float om, float os) {
        const float n = fmaxf(m, om), b = n == NEG_INF ? 0.0f : n;
        s = s * __expf(m - b) + os * __expf(om - b);
        m = n;
    };
    for (int64_t k = tid >> 4; k < a.chunks; k += 4 * LSE_LANES) {
        f32x2_t p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t c = k + i * LSE_LANES;
            p[i] = a.part[min(c, a.chunks - 1) * a.tp + t];
            if (c >= a.chunks) p[i] = f32x2_t{NEG_INF, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < 4; i++) add(p[i].x, p[i].y);
    }
    for (int w = LSE_LANES; w > 1; w /= 2) {
        s_p[tid >> 4][tl] = f32x2_t{m, s};
        __syncthreads();
        if ((tid >> 4) < w / 2) add(s_p[(tid >> 4) + w / 2][tl].x, s_p[(tid >> 4) + w / 2][tl].y);
        __syncthreads();
    }
    if (tid >= 16 || t >= a.tokens) return;
    const float lse = m + logf(s);
    const int64_t v = target_of(a.target, t, a.ignore, a.rows);
    a.lse[t] = lse;
    a.loss[t] = v == TARGET_SKIP ? 0.0f : v == TARGET_BAD ? __builtin_nanf("") : lse - a.at[t];
}

struct DxArgs {
    const f32x4_t* part;  // of GradEpi
    int slices, tp, n, tokens;
    int64_t np;
    DxFactor fac;
    void* dx;
    int dx_dt;
};
// A wave 16 tokens by 128 columns, a lane 4 runs of 8 neighbouring columns.
// SPLIT: the 4 waves of a workgroup take the slices in turn and meet in LDS
// (8 slices of 200 x 2048 sums: 8.4 us without, 5.0).
template <bool SPLIT>
__global__ void __launch_bounds__(256) dx_kernel(const DxArgs a)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, tile = blockIdx.y, t = tile * 16 + (lane & 15);
    const int64_t g = SPLIT ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (!SPLIT && g * 128 >= a.n) return;
    DxFactor fac = a.fac;
    fac.init();
    f32x4_t v[8];
    const f32x4_t* p = a.part + ((int64_t)tile * (a.np / 128) + g) * 512 + lane;
    const int64_t ld = (int64_t)(a.tp / 16) * (a.np / 128) * 512;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = p[(SPLIT ? wave : 0) * ld + i * 64];
    for (int z = SPLIT ? wave + 4 : 1; z < a.slices; z += SPLIT ? 4 : 1)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += p[z * ld + i * 64];
    if constexpr (SPLIT) {
        __shared__ f32x4_t s_v[4][8][64];
#pragma unroll
        for (int i = 0; i < 8; i++) s_v[wave][i][lane] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (the wave finishes element `wave` of every lane)
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) s += ((const float*)&s_v[w][i][lane])[wave];
            v[i][0] = s;
        }
    }
    if (t >= a.tokens) return;
    const DxFactor::Of f = fac.of(t);
#pragma unroll
    for (int e = 0; e < (SPLIT ? 1 : 4); e++) {
        const int64_t col = g * 128 + (q * 4 + (SPLIT ? wave : e)) * 8;
        if (col < a.n) store_run(a.dx, a.dx_dt, (int64_t)t * a.n + col, v, e, f);
    }
}

struct DsArgs {
    MatArgs m;
    const float* part;  // [chunks][ld]
    int chunks;
    int64_t ld;
    float rs;
    float* ds[2];
    int add;
};
// 32 rows a workgroup, 8 threads a row over the chunks
__global__ void __launch_bounds__(256) ds_kernel(const DsArgs a)
{
    __shared__ float s_s[8][32];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t p = (int64_t)blockIdx.x * 32 + x;  // (a whole number of workgroups)
    float s = 0.0f;
#pragma unroll 8
    for (int k = y; k < a.chunks; k += 8) s += a.part[k * a.ld + p];
    s_s[y][x] = s;
    __syncthreads();
    if (y) return;
    int mat;
    const int64_t row = mat_row(a.m, p >> 4, (int)(p & 15), mat);
    if (row >= a.m.rows) return;
#pragma unroll
    for (int k = 1; k < 8; k++) s += s_s[k][x];
    float* d = a.ds[mat] + row;
    *d = (a.add ? *d : 0.0f) + s * a.rs;
}

__global__ void __launch_bounds__(256) zero_kernel(float* p, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0.0f;
}

// ------------------------------------------------------------------- host
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct Bump {
    size_t at = 0;
    size_t take(size_t bytes)
    {
        const size_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    }
};

// Tokens are taken PANEL_TOKENS at a time, and the matrix in pieces whose
// panel of gradients (2 bytes a token and row) stays near PIECE_BYTES.
constexpr int64_t PANEL_TOKENS = 8192;
constexpr int64_t PIECE_BYTES = 128 << 20;
constexpr int64_t PIECE_MAX_ROWS = 16384, PIECE_MIN_ROWS = 4096, PIECE_FORWARD_ROWS = 32768;

// few_kernel: up to here it reads 16-bit rows as they are.  A lane's 8 loads are
// a line each; 16 tokens of a 151936-row head took 245 us so, 48 packed ones 215.
bool few_own(int64_t tokens, int x_dt) { return tokens <= 4 && x_dt <= VQ2_DT_BF16; }

int64_t few_pairs(const PanelCall& c) { return ((c.rows + 15) / 16 * c.nmat + 1) / 2; }

// Its token tiles a workgroup, and whether a wave of 128 tokens has its rows to
// itself.
int few_tiles(int64_t tokens)
{
    if (tokens <= 64) return tokens <= 16 ? 1 : tokens <= 32 ? 2 : 4;
    return tokens <= (tokens + 127) / 128 * 96 ? 6 : 8;  // as many blocks as of 8, but no larger than they have to be
}
bool few_alone(int tt, int64_t pairs) { return tt >= 6 && pairs >= 1024; }

// Its workgroups along the pairs of tiles: for the loss as many as are
// resident, each keeps running sums over its pairs.
int few_groups(const PanelCall& c, int64_t tokens)
{
    const int tt = few_tiles(tokens);
    const int64_t pairs = few_pairs(c), units = few_alone(tt, pairs) ? (pairs + 3) / 4 : pairs;
    if (c.what != PANEL_STATS) return (int)units;
    return (int)std::min<int64_t>(units, (int64_t)device_cu_count() * (tt >= 6 || few_own(tokens, c.x_dt) ? 2 : 3));
}

// Whether few_kernel is ahead of panels: it gathers every centroid once for
// each block of 128 tokens, panels once, but they store and read it again, and
// take two launches more.  In gathers: a block costs them and 10^5, panels 1.3
// times as many and 2.8 * 10^6.  Measured (us a call; codes of the call, tokens: few /
// panels): 65 k, 512 15 / 24; 262 k, 1024 31 / 39, 2048 45 / 42; 512 k, 333 25 / 37, 1024 43 / 41;
// 3.1 M, 128 33 / 51, 256 54 / 52, 512 96 / 59; 6.3 M, 128 51 / 61, 192 82 / 62; 12.9 M, 128
// 108 / 128, 160 190 / 140; 38.9 M, 1 171 / 335, 128 270 / 335, 160 478 / 367.
bool few_ahead(const PanelCall& c, int64_t tokens)
{
    if (c.cb_dt == VQ2_DT_F32) return false;  // (its centroids would take two products each)
    const double gathers = (double)c.rows * c.nmat * (double)(c.n / 8) * (c.s2 == VQ2_S2_U16 ? 2 : 1);
    const double blocks = (double)((tokens + 127) / 128);
    return tokens <= 64 || blocks * (gathers + 1e5) <= 1.3 * gathers + 2.8e6;
}

struct Plan {
    int64_t chunk;       // tokens of a chunk (the last may be shorter)
    int64_t tp;          // of them, padded
    int64_t tiles;       // 16-row tiles of all matrices, padded to whole workgroups
    int64_t piece;       // tiles of a piece
    bool direct;         // the gradient's product writes dx
    bool few[2];         // few_kernel for a whole chunk, and for the last one
    int mt, gmt;         // tiles of a wave: the first product's, the gradient's
    int tops;            // workgroups of prep_scales
    int books;           // of book_max
    int parts, tparts, kt;  // parts of a weight in the rows' panel, and the columns'
    int64_t np;          // columns, padded
    int slices;
    size_t fac, top, book, sc, xp, w, wt, p, acc, stats, at, ds, dfac, total;
};

enum { STATS = PANEL_STATS, DLOGIT = PANEL_DLOGIT, GATED = PANEL_GATED, DGATED = PANEL_DGATED, PRODUCT = PANEL_PRODUCT };

// values of a stage's codebook
int64_t book_values(const PanelCall& c, int stage)
{
    return stage == 0 || c.s2 == VQ2_S2_U16 ? 65536 * 8 : c.s2 == VQ2_S2_U8 ? 256 * 8 : 0;
}

Plan plan_of(const PanelCall& c)
{
    Plan p{};
    const bool grad = c.what == DLOGIT || c.what == DGATED || c.what == PRODUCT;
    p.chunk = std::min(c.tokens, PANEL_TOKENS);
    p.tp = up(p.chunk, PG_N);
    p.tiles = up((c.rows + 15) / 16 * c.nmat, pg_m(8) / 16);
    p.kt = (int)(c.n / 32);
    // (each chunk as a call of its own would take it)
    const int64_t rest = c.tokens % p.chunk;
    p.few[0] = !grad && few_ahead(c, p.chunk);
    p.few[1] = rest ? !grad && few_ahead(c, rest) : p.few[0];
    const bool exact = c.cb_dt != VQ2_DT_F32 && c.s2 == VQ2_S2_NONE;
    const bool fine = c.y_dt != VQ2_DT_BF16;
    const bool wide = c.what == STATS || c.what == DLOGIT || c.ds[0] != nullptr || fine;
    p.parts = !exact && wide ? 2 : 1;
    p.tparts = !exact && fine ? 2 : 1;
    int64_t rows = grad ? PIECE_MAX_ROWS : PIECE_FORWARD_ROWS;
    while (grad && rows > PIECE_MIN_ROWS && rows * p.tp * 2 > PIECE_BYTES) rows /= 2;
    p.piece = std::min(p.tiles, rows / 16);
    p.np = up(c.n, pg_m(8));
    p.slices = 1;
    // Wave tiles of 128 rows, two workgroups a CU, where that many are there;
    // of 64 otherwise, which keep up with them three a CU.
    const int64_t slots = 2 * (int64_t)device_cu_count();
    p.mt = p.piece * 16 / pg_m(8) * (p.tp / PG_N) >= slots ? 8 : 4;
    Bump b;
    p.fac = b.take(p.tp * 4);
    p.tops = (int)((p.tiles * 16 + PREP_ROWS - 1) / PREP_ROWS);
    p.top = b.take(p.tops * 4);
    p.books = c.what == DGATED ? (int)((book_values(c, 0) + book_values(c, 1) + BOOK_VALUES - 1) / BOOK_VALUES) : 0;
    p.book = b.take(p.books * 4);
    p.sc = b.take(p.tiles * 16 * 4);
    p.xp = b.take(p.tp * c.n * 2);
    // (none of a matrix is kept where few_kernel takes all chunks: one token's loss over 151936 x 2048 had 134 MB)
    const bool w = grad ? c.what != PRODUCT || c.ds[0] : !p.few[0] || !p.few[1];
    p.w = b.take(w ? p.piece * 16 * c.n * 2 * p.parts : 0);
    if (grad) {
        p.wt = b.take(p.piece * 16 * p.np * 2 * p.tparts);
        p.p = b.take(p.piece * 16 * p.tp * 2);
        // As few slices of a piece's rows as fill the device (each adds a pass
        // over the sums), of at least 8 k tiles.
        const int64_t wg = p.np / pg_m(8) * (p.tp / PG_N), most = std::max<int64_t>(1, p.piece / 2 / 8);
        // One piece in one slice is written as dx at once.
        const bool one = p.piece == p.tiles;
        p.gmt = 2 * wg >= slots ? 8 : 4;
        while (p.slices < 64 && wg * (8 / p.gmt) * p.slices < slots && p.slices * 2 <= most) p.slices *= 2;
        p.direct = one && p.slices == 1;
        p.acc = b.take(p.direct ? 0 : p.slices * p.tp * p.np * 4);
        if (c.ds[0]) p.ds = b.take(p.tp / (16 * PG_NT) * p.tiles * 16 * 4);
        if (c.what != DLOGIT) p.dfac = b.take(p.tp * 4);
    }
    if (c.what == STATS) {
        // parts: a wave's rows, or (few_kernel) a workgroup's, or a wave's
        p.stats = b.take(std::max<int64_t>(p.tiles / 4, p.few[0] || p.few[1] ? 12 * device_cu_count() : 0) * p.tp * 8);
        p.at = b.take(p.tp * 4);
    }
    p.total = b.at;
    return p;
}

template <int MT, class Epi>
hipError_t gemm_typed(const PanelGemmArgs& g, const Epi& e, int64_t tile0, hipStream_t st)
{
    static std::once_flag once;
    static hipError_t attr = hipSuccess;
    std::call_once(once, [] {
        attr = hipFuncSetAttribute((const void*)panel_gemm_kernel<MT, Epi>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   pg_lds(MT));
    });
    if (attr != hipSuccess) return attr;
    hipLaunchKernelGGL((panel_gemm_kernel<MT, Epi>), dim3((unsigned)(g.gm * g.gn * g.gz)), dim3(PG_THREADS),
                       pg_lds(MT), st, g, e, tile0);
    return hipGetLastError();
}

// rows of panel a in g.gm * pg_m(8)
template <class Epi>
hipError_t gemm(PanelGemmArgs g, int mt, const Epi& e, int64_t tile0, hipStream_t st)
{
    if (mt == 8) return gemm_typed<8>(g, e, tile0, st);
    g.gm *= 2;
    return gemm_typed<4>(g, e, tile0, st);
}

template <int CBT, int S2, int WP, int TP>
hipError_t dequant_parts(const DequantArgs& a, int64_t tiles, hipStream_t st)
{
    if constexpr (TP == 0)
        hipLaunchKernelGGL((dequant_plain_kernel<CBT, S2, WP>), dim3((unsigned)(tiles / 4), (unsigned)((a.m.ng / 4 + 7) / 8)),
                           dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((dequant_both_kernel<CBT, S2, WP, TP>), dim3((unsigned)(tiles / 8), (unsigned)((a.m.ng + 15) / 16)),
                           dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int CBT, int S2>
hipError_t dequant_typed(const DequantArgs& a, int wp, int tp, int64_t tiles, hipStream_t st)
{
    constexpr bool EXACT = CBT != VQ2_DT_F32 && S2 == VQ2_S2_NONE;
    if constexpr (!EXACT) {
        if (tp == 0 && wp == 2) return dequant_parts<CBT, S2, 2, 0>(a, tiles, st);
        if (tp == 2 && wp == 0) return dequant_parts<CBT, S2, 0, 2>(a, tiles, st);
        if (tp == 2) return dequant_parts<CBT, S2, 2, 2>(a, tiles, st);
        if (wp == 2) return dequant_parts<CBT, S2, 2, 1>(a, tiles, st);
    }
    if (tp == 0) return dequant_parts<CBT, S2, 1, 0>(a, tiles, st);
    if (wp == 0) return dequant_parts<CBT, S2, 0, 1>(a, tiles, st);
    return dequant_parts<CBT, S2, 1, 1>(a, tiles, st);
}

template <int CBT>
hipError_t dequant_s2(const DequantArgs& a, int s2, int wp, int tp, int64_t tiles, hipStream_t st)
{
    if (s2 == VQ2_S2_NONE) return dequant_typed<CBT, VQ2_S2_NONE>(a, wp, tp, tiles, st);
    if (s2 == VQ2_S2_U8) return dequant_typed<CBT, VQ2_S2_U8>(a, wp, tp, tiles, st);
    return dequant_typed<CBT, VQ2_S2_U16>(a, wp, tp, tiles, st);
}

// wp, tp: parts of the rows' and the columns' panel, 0 for none
hipError_t dequant(const DequantArgs& a, int cb_dt, int s2, int wp, int tp, int64_t tiles, hipStream_t st)
{
    if (cb_dt == VQ2_DT_F16) return dequant_s2<VQ2_DT_F16>(a, s2, wp, tp, tiles, st);
    if (cb_dt == VQ2_DT_BF16) return dequant_s2<VQ2_DT_BF16>(a, s2, wp, tp, tiles, st);
    return dequant_s2<VQ2_DT_F32>(a, s2, wp, tp, tiles, st);
}

template <int CBT, int S2, class Epi>
hipError_t few_typed(const FewArgs& a, const Epi& e, int tt, int groups, hipStream_t st)
{
    const dim3 grid((unsigned)groups, (unsigned)((a.tokens + 16 * tt - 1) / (16 * tt))), block(256);
    if (tt == 1 && few_own(a.tokens, a.x_dt)) hipLaunchKernelGGL((few_kernel<CBT, S2, 1, 4, true, Epi>), grid, block, 0, st, a, e);
    else if (tt == 1) hipLaunchKernelGGL((few_kernel<CBT, S2, 1, 4, false, Epi>), grid, block, 0, st, a, e);
    else if (tt == 2) hipLaunchKernelGGL((few_kernel<CBT, S2, 2, 4, false, Epi>), grid, block, 0, st, a, e);
    else if (tt == 4) hipLaunchKernelGGL((few_kernel<CBT, S2, 4, 4, false, Epi>), grid, block, 0, st, a, e);
    else if (few_alone(tt, a.pairs)) {
        if (tt == 6) hipLaunchKernelGGL((few_kernel<CBT, S2, 6, 1, false, Epi>), grid, block, 0, st, a, e);
        else hipLaunchKernelGGL((few_kernel<CBT, S2, 8, 1, false, Epi>), grid, block, 0, st, a, e);
    } else {
        if (tt == 6) hipLaunchKernelGGL((few_kernel<CBT, S2, 6, 4, false, Epi>), grid, block, 0, st, a, e);
        else hipLaunchKernelGGL((few_kernel<CBT, S2, 8, 4, false, Epi>), grid, block, 0, st, a, e);
    }
    return hipGetLastError();
}

template <class Epi>
hipError_t few(const FewArgs& a, const Epi& e, int tt, int groups, int cb_dt, int s2, hipStream_t st)
{
    if (cb_dt == VQ2_DT_F16) {
        if (s2 == VQ2_S2_NONE) return few_typed<VQ2_DT_F16, VQ2_S2_NONE>(a, e, tt, groups, st);
        if (s2 == VQ2_S2_U8) return few_typed<VQ2_DT_F16, VQ2_S2_U8>(a, e, tt, groups, st);
        return few_typed<VQ2_DT_F16, VQ2_S2_U16>(a, e, tt, groups, st);
    }
    if (s2 == VQ2_S2_NONE) return few_typed<VQ2_DT_BF16, VQ2_S2_NONE>(a, e, tt, groups, st);
    if (s2 == VQ2_S2_U8) return few_typed<VQ2_DT_BF16, VQ2_S2_U8>(a, e, tt, groups, st);
    return few_typed<VQ2_DT_BF16, VQ2_S2_U16>(a, e, tt, groups, st);
}

}  // namespace

size_t panel_workspace_bytes(const PanelCall& c) { return c.tokens ? plan_of(c).total : 0; }

#define TRY(call)                                               \
    do {                                                        \
        const hipError_t e_ = (call);                           \
        if (e_ != hipSuccess) return set_hip_error(e_, c.who);  \
    } while (0)

int panel_launch(const PanelCall& c)
{
    const hipStream_t st = (hipStream_t)c.stream;
    const MatArgs mats{{{c.mat[0].i0, c.mat[0].i1, c.mat[0].scale}, {c.mat[1].i0, c.mat[1].i1, c.mat[1].scale}},
                       c.nmat, c.rows, (int)(c.n / 8), c.s_dt, c.cb0, c.cb1};
    if (c.tokens == 0) {
        for (int k = 0; k < c.nmat; k++)
            if (c.ds[k]) {
                hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((c.rows + 255) / 256)), dim3(256), 0, st, c.ds[k], c.rows);
                TRY(hipGetLastError());
            }
        return VQ2_OK;
    }
    const Plan p = plan_of(c);
    bool aligned = true;  // (rows are n / 8 codes, a multiple of 8)
    for (int k = 0; k < c.nmat; k++) aligned = aligned && (uintptr_t)c.mat[k].i0 % 16 == 0 && (uintptr_t)c.mat[k].i1 % 16 == 0;
    char* ws = (char*)c.workspace;
    const bool grad = c.what == DLOGIT || c.what == DGATED || c.what == PRODUCT;
    const bool first = c.what != PRODUCT || c.ds[0];  // the product of weights and tokens
    float* fac = (float*)(ws + p.fac);
    float* top = (float*)(ws + p.top);
    const RowTop amax{top, p.tops};
    float* sc = (float*)(ws + p.sc);
    half8_t* xp = (half8_t*)(ws + p.xp);
    half8_t* w = first ? (half8_t*)(ws + p.w) : nullptr;
    half8_t* wt = grad ? (half8_t*)(ws + p.wt) : nullptr;
    half8_t* pp = (half8_t*)(ws + p.p);
    f32x4_t* acc = (f32x4_t*)(ws + p.acc);
    float* ds = c.ds[0] ? (float*)(ws + p.ds) : nullptr;
    float* dfac = (float*)(ws + p.dfac);
    BlockBound bound{amax, {(const float*)(ws + p.book), p.books}, fac, 0};
    if (c.what == DGATED) {
        int lg = 0;
        while ((int64_t)1 << lg < c.n) lg++;
        bound.bits = 14 + lg + 1 + (c.s2 != VQ2_S2_NONE);
    }
    bool prepared = false;  // the row scales
    const int64_t xsize = c.x_dt == VQ2_DT_F32 ? 4 : c.x_dt <= VQ2_DT_BF16 ? 2 : 1;
    for (int64_t t0 = 0; t0 < c.tokens; t0 += p.chunk) {
        const int tokens = (int)std::min(p.chunk, c.tokens - t0);
        const int tp = (int)up(tokens, PG_N);
        const int64_t ds_ld = p.tiles * 16;
        const bool few_call = p.few[tokens < p.chunk];
        const void* dy = c.dy ? (const char*)c.dy + t0 * c.rows * dt_size(c.dy_dt) : nullptr;
        const int64_t* target = c.target ? c.target + t0 : nullptr;
        const int dy_vec = dy && c.rows % 8 == 0 && (uintptr_t)dy % 16 == 0;
        void* dx = c.y && grad ? (char*)c.y + t0 * c.n * dt_size(c.y_dt) : nullptr;
        const DxFactor dxf{amax, c.what == DLOGIT ? nullptr : dfac, c.dloss ? c.dloss + t0 : nullptr, target, c.rows, c.ignore, bound, 0};
        const bool dy32 = c.dy_dt == VQ2_DT_F32, fours = c.rows % 4 == 0 && (uintptr_t)dy % (dy32 ? 16 : 8) == 0;
        const UpstreamArgs upstream{dy, c.dy_dt, tokens, fours, c.rows};
        const bool v16 = fours && !dy32;
        const bool prep = !few_call && !prepared;
        prepared = prepared || prep;
        const PrologueArgs pro{
            PackArgs{(const char*)c.x + t0 * c.n * xsize, c.x_dt, tokens, (int)c.n, c.x_scale ? c.x_scale + t0 : nullptr,
                     c.what == DLOGIT ? target : nullptr, c.ignore, xp, fac,
                     first && !(few_call && few_own(tokens, c.x_dt)) ? tp / 16 : 0},
            DyMaxArgs{dy, c.dy_dt, tokens, dy_vec, c.rows, dfac,
                      c.what == DGATED || c.what == PRODUCT ? tp / 16 : 0},
            PrepArgs{mats, c.rs, ds_ld, sc, top, prep ? p.tops : 0},
            BookArgs{{c.cb0, c.cb1}, c.cb_dt, (int)(book_values(c, 0) / BOOK_VALUES), {book_values(c, 0), book_values(c, 1)},
                     (float*)(ws + p.book), prep ? p.books : 0}};
        if (const int groups = pro.pack.tiles + pro.dy.groups + pro.prep.groups + pro.book.groups) {
            hipLaunchKernelGGL(prologue_kernel, dim3((unsigned)groups), dim3(64 * PK_WAVES), 0, st, pro);
            TRY(hipGetLastError());
        }
        auto lse_launch = [&](int64_t chunks) {
            hipLaunchKernelGGL(lse_kernel, dim3((unsigned)((tokens + 15) / 16)), dim3(16 * LSE_LANES), 0, st,
                               LseArgs{(const f32x2_t*)(ws + p.stats), chunks, tokens, tp, target, c.rows, c.ignore,
                                       (const float*)(ws + p.at), c.loss + t0, c.lse_out + t0});
            return hipGetLastError();
        };
        const StatsEpi stats{sc, fac, target, c.rows, c.ignore, tokens, tp, (f32x2_t*)(ws + p.stats), (float*)(ws + p.at)};
        const GatedEpi gated{sc, fac, c.y && !grad ? (char*)c.y + t0 * c.rows * dt_size(c.y_dt) : nullptr, c.y_dt, tokens, c.rows,
                             c.rows % 4 == 0 && (uintptr_t)c.y % 16 == 0, c.act};
        if (few_call) {
            const FewArgs f{mats, few_pairs(c), xp, fac, (const char*)c.x + t0 * c.n * xsize, c.x_dt, tokens, (int)c.n,
                            c.rs};
            const int tt = few_tiles(tokens), groups = few_groups(c, tokens);
            if (c.what == GATED) {
                TRY(few(f, gated, tt, groups, c.cb_dt, c.s2, st));
            } else {
                TRY(few(f, stats, tt, groups, c.cb_dt, c.s2, st));
                TRY(lse_launch(few_alone(tt, few_pairs(c)) ? groups * 4 : groups));
            }
            continue;
        }
        for (int64_t tile0 = 0; tile0 < p.tiles; tile0 += p.piece) {
            const int64_t tiles = std::min(p.piece, p.tiles - tile0);
            const int vkt = (int)(tiles / 2);
            TRY(dequant(DequantArgs{mats, tile0, w, wt, vkt, aligned}, c.cb_dt, c.s2, w ? p.parts : 0, wt ? p.tparts : 0, tiles, st));
            const PanelGemmArgs g{w, xp, p.parts * p.kt, p.kt, (int)(tiles * 16 / pg_m(8)), tp / PG_N, 1};
            if (c.what == STATS)
                TRY(gemm(g, p.mt, stats, tile0, st));
            else if (c.what == GATED)
                TRY(gemm(g, p.mt, gated, tile0, st));
            else if (c.what == DLOGIT)
                TRY(gemm(g, p.mt, DlogitEpi{sc, fac, c.lse + t0, c.dloss + t0, target, amax, c.rows, c.ignore, tile0, tokens, tp, vkt,
                                          pp, ds, ds_ld}, tile0, st));
            else if (c.what == DGATED && v16)
                TRY(gemm(g, p.mt, DgatedEpi<true>{sc, fac, dfac, {upstream}, bound, tp, vkt, tile0, pp, ds, ds_ld, c.act}, tile0, st));
            else if (c.what == DGATED)
                TRY(gemm(g, p.mt, DgatedEpi<false>{sc, fac, dfac, {upstream}, bound, tp, vkt, tile0, pp, ds, ds_ld, c.act}, tile0, st));
            else if (first && v16)
                TRY(gemm(g, p.mt, ColsumEpi<true>{fac, {upstream}, ds, ds_ld}, tile0, st));
            else if (first)
                TRY(gemm(g, p.mt, ColsumEpi<false>{fac, {upstream}, ds, ds_ld}, tile0, st));
            if (!grad) continue;
            if (c.what == PRODUCT) {
                const dim3 grid((unsigned)(tp / 16), (unsigned)((vkt + 15) / 16));
                if (v16)
                    hipLaunchKernelGGL(dy_panel_kernel<true>, grid, dim3(256), 0, st,
                                       DyArgs<true>{{upstream}, tile0 * 16, sc, amax, dfac, pp, vkt});
                else
                    hipLaunchKernelGGL(dy_panel_kernel<false>, grid, dim3(256), 0, st,
                                       DyArgs<false>{{upstream}, tile0 * 16, sc, amax, dfac, pp, vkt});
                TRY(hipGetLastError());
            }
            const int slices = (int)std::min<int64_t>(p.slices, vkt);
            const PanelGemmArgs g2{wt, pp, p.tparts * vkt, vkt, (int)(p.np / pg_m(8)), tp / PG_N, slices};
            TRY(gemm(g2, p.gmt, GradEpi{acc, p.np, tp, tile0 != 0, p.direct ? dx : nullptr, c.y_dt, tokens, (int)c.n, dxf}, 0, st));
        }
        if (c.what == STATS) TRY(lse_launch(p.tiles / p.mt));
        if (!grad) continue;
        if (!p.direct) {
            const DxArgs d{acc, p.slices, tp, (int)c.n, tokens, p.np, dxf, dx, c.y_dt};
            const unsigned rows = (unsigned)((tokens + 15) / 16);
            if (p.slices >= 4) hipLaunchKernelGGL(dx_kernel<true>, dim3((unsigned)((c.n + 127) / 128), rows), dim3(256), 0, st, d);
            else hipLaunchKernelGGL(dx_kernel<false>, dim3((unsigned)((c.n + 511) / 512), rows), dim3(256), 0, st, d);
            TRY(hipGetLastError());
        }
        if (ds) {
            hipLaunchKernelGGL(ds_kernel, dim3((unsigned)(ds_ld / 32)), dim3(256), 0, st,
                               DsArgs{mats, ds, tp / (16 * PG_NT), ds_ld, c.rs, {c.ds[0], c.ds[1]}, t0 != 0});
            TRY(hipGetLastError());
        }
    }
    return VQ2_OK;
}

}  // namespace vq2
