// vq2_norm.hip -- the norm in front of packed products: residual addition,
// root mean square, weight, and the rotation the product wants, in one pass
// over the rows; and its backward pass.
//
//   h = x + residual,  r = (mean(h^2) + eps)^-1/2,  u = h r w
//   y = u, or R u with R = blockdiag(H_hb) S P scale (vq2_rht), in 16 or 32 bits,
//       or in 8 bits under a scale for each row
//
//   g = R^T dy,  dx = dh + r g w - h r^3 mean(g w h),  dw = sum over rows of g h r
//
// Bound by HBM: every element is read once and written once, the row stays in
// registers between.  16384 rows of 2048 (bf16, residual: 268 MB) 41.5 us, 6.5 TB/s;
// rotated 51; backward 42, rotated 67.  Rows that are no multiple of 8 values are loaded one
// by one (16000 x 2047: 49 us).  A thread holds 8 neighbouring values (16-byte loads) of each
// 2048: the transform's first 3 stages are in its registers, the next 6 are
// exchanges between lanes, the ones above one pass through LDS between the waves
// of a row, and what is left in registers again.  The permutation goes through
// LDS, too.  A workgroup takes rows in turn, the next one's loads ahead, and
// loads its part of the weights and tables once.  All arithmetic is fp32; h is
// rounded where it is stored, y is made from the unrounded sum.
#include <algorithm>
#include <type_traits>

#include "vq2_internal.hpp"
#include "vq2_panel.hpp"

namespace vq2 {

namespace {

// Threads of a workgroup: 256, or backward 512 that share one row above 6144
// values (4096 x 8192: 95 us; with 256, 32 values a thread, 184, spilled.
// Forward 256 threads take 65 us, 512 87).
constexpr int threads_of(int TPR) { return TPR > 256 ? TPR : 256; }

// lane i <- lane i ^ 4, i ^ 8 within a row of 16
__device__ __forceinline__ float dpp_xor4(float v)
{
    // row_half_mirror is i ^ 7, quad_perm [3,2,1,0] i ^ 3
    return __int_as_float(dpp_mov<0x1B>(dpp_mov<0x141>(__float_as_int(v))));
}
__device__ __forceinline__ float dpp_xor8(float v) { return __int_as_float(dpp_mov<0x128>(__float_as_int(v))); }  // row_ror:8

// One butterfly stage between lanes: the lane whose bit is clear takes the
// sum, the other the difference (two instructions a value: the exchange is
// part of the addition).
template <class X>
__device__ __forceinline__ void lane_stage(float (&v)[8], bool high, X other)
{
    const float s = high ? -1.0f : 1.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float t = v[k] * s;
        v[k] = other(v[k]) + t;
    }
}
// Between rows of 16 lanes (STEP 16) or halves of the wave (32), two values
// at a time: a swap brings both partners of one value into one lane, and
// another puts the results back.
template <int STEP>
__device__ __forceinline__ void swap2(float& a, float& b)
{
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    const auto r = STEP == 16 ? __builtin_amdgcn_permlane16_swap(x, y, false, false)
                              : __builtin_amdgcn_permlane32_swap(x, y, false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
template <int STEP>
__device__ __forceinline__ void swap_stage(float (&v)[8])
{
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        swap2<STEP>(v[k], v[k + 1]);
        const float s = v[k] + v[k + 1], d = v[k] - v[k + 1];
        v[k] = s;
        v[k + 1] = d;
        swap2<STEP>(v[k], v[k + 1]);
    }
}

// Hadamard transform of blocks of hb values; the row's value 8 (c TPR + id) + k
// is v[c][k] of its thread id.  s: V * 8 * TPR floats of the row.
template <int V, int TPR>
__device__ __forceinline__ void hadamard(float (&v)[V][8], int hb, int id, float* s)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < V; c++) {
#pragma unroll
        for (int st = 1; st < 8; st *= 2)
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (!(k & st)) {
                    const float a = v[c][k], b = v[c][k + st];
                    v[c][k] = a + b;
                    v[c][k + st] = a - b;
                }
        // (blocks have 64 values or more)
        lane_stage(v[c], lane & 1, [](float a) { return dpp_xor1(a); });
        lane_stage(v[c], lane & 2, [](float a) { return dpp_xor2(a); });
        lane_stage(v[c], lane & 4, [](float a) { return dpp_xor4(a); });
    }
    if (hb >= 128)
#pragma unroll
        for (int c = 0; c < V; c++) lane_stage(v[c], lane & 8, [](float a) { return dpp_xor8(a); });
    if (hb >= 256)
#pragma unroll
        for (int c = 0; c < V; c++) swap_stage<16>(v[c]);
    if (hb >= 512)
#pragma unroll
        for (int c = 0; c < V; c++) swap_stage<32>(v[c]);
    if (TPR <= 64 || hb < 1024) return;
    // between the waves of a row: that of wave w is the sum over the m of its
    // block of +- theirs, minus where w and the other share an odd number of bits
    const int w = id >> 6;
    f32x4_t* p = (f32x4_t*)s;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < V; c++) {
        p[(c * 2 + 0) * TPR + id] = f32x4_t{v[c][0], v[c][1], v[c][2], v[c][3]};
        p[(c * 2 + 1) * TPR + id] = f32x4_t{v[c][4], v[c][5], v[c][6], v[c][7]};
    }
    __syncthreads();
    auto exchange = [&](auto count) {
        constexpr int M = decltype(count)::value;
        float sg[M];
#pragma unroll
        for (int j = 0; j < M; j++) sg[j] = __builtin_popcount(w & j) & 1 ? -1.0f : 1.0f;
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f32x4_t* q = p + (c * 2 + h) * TPR + (w & ~(M - 1)) * 64 + (id & 63);
                f32x4_t o = q[0];
#pragma unroll
                for (int j = 1; j < M; j++) o += q[j * 64] * sg[j];
#pragma unroll
                for (int k = 0; k < 4; k++) v[c][4 * h + k] = o[k];
            }
    };
    if (hb == 1024) exchange(std::integral_constant<int, 2>());
    else if (TPR == 256 || hb == 2048) {
        if constexpr (TPR >= 256) exchange(std::integral_constant<int, 4>());
    } else {
        if constexpr (TPR >= 512) exchange(std::integral_constant<int, 8>());
    }
    // blocks above 8 TPR: between a thread's own parts
#pragma unroll
    for (int st = 1; st < V; st *= 2) {
        if (hb < 16 * TPR * st) break;
#pragma unroll
        for (int c = 0; c < V; c++)
            if (!(c & st) && c + st < V)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float a = v[c][k], b = v[c + st][k];
                    v[c][k] = a + b;
                    v[c + st][k] = a - b;
                }
    }
}

// N values that every thread of the row has a part of; s: N words for each
// wave of the workgroup
template <int TPR, int N, class Op>
__device__ __forceinline__ void row_reduce(float (&v)[N], float* s, Op op)
{
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = op(v[i], dpp_xor1(v[i]));
        v[i] = op(v[i], dpp_xor2(v[i]));
        v[i] = op(v[i], dpp_half_mirror(v[i]));
        v[i] = op(v[i], dpp_row_mirror(v[i]));
        if (TPR >= 64) {
            v[i] = op(v[i], swz_xor16(v[i]));
            v[i] = op(v[i], xor32(v[i]));
        }
    }
    if (TPR <= 64) return;
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    __syncthreads();  // (the last call's values have been read)
#pragma unroll
    for (int i = 0; i < N; i++)
        if ((threadIdx.x & 63) == 0) s[i * 8 + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = s[i * 8 + first];
#pragma unroll
        for (int k = 1; k < W; k++) v[i] = op(v[i], s[i * 8 + first + k]);
    }
}
__device__ __forceinline__ float add_op(float a, float b) { return a + b; }
// maximum of magnitudes by their bits: a NaN is above everything and stays
__device__ __forceinline__ float bits_op(float a, float b)
{
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// A thread's part of a row.  VEC: 8 neighbouring values in each of the V parts,
// by 16-byte accesses; otherwise value (8 c + k) TPR + id, one by one.
template <int V, int TPR, bool VEC>
__device__ __forceinline__ int place(int c, int k, int id)
{
    return VEC ? (c * TPR + id) * 8 + k : (c * 8 + k) * TPR + id;
}

// A row's values as they are loaded (VEC: 16 or 32 bytes of type DT; else a word
// each), and as numbers.  No load is behind a branch: past the row's end the
// first value is loaded, and dropped.
template <int DT, int V, bool VEC>
struct Raw {
    u32x4 w[V][VEC && DT != VQ2_DT_F32 ? 1 : 2];
};
template <int DT, int V, int TPR, bool VEC>
__device__ __forceinline__ void load_raw(Raw<DT, V, VEC>& r, const void* p, int64_t row, int n, int id)
{
    const char* base = (const char*)p + row * n * (DT == VQ2_DT_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < V; c++) {
        if constexpr (VEC) {
            const int i = place<V, TPR, VEC>(c, 0, id);
            constexpr int N = DT == VQ2_DT_F32 ? 2 : 1;
            const u32x4* q = (const u32x4*)(base + (i < n ? i : 0) * (DT == VQ2_DT_F32 ? 4 : 2));
#pragma unroll
            for (int k = 0; k < N; k++) r.w[c][k] = q[k];
            if (i >= n)
#pragma unroll
                for (int k = 0; k < N; k++) r.w[c][k] = u32x4{0, 0, 0, 0};
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = place<V, TPR, VEC>(c, k, id), at = i < n ? i : 0;
                r.w[c][k / 4][k % 4] = DT == VQ2_DT_F32 ? ((const uint32_t*)base)[at] : (uint32_t)((const uint16_t*)base)[at];
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (place<V, TPR, VEC>(c, k, id) >= n) r.w[c][k / 4][k % 4] = 0;
        }
    }
}
template <int DT, int V, bool VEC>
__device__ __forceinline__ void numbers(float (&v)[V][8], const Raw<DT, V, VEC>& r)
{
#pragma unroll
    for (int c = 0; c < V; c++) {
        if constexpr (!VEC || DT == VQ2_DT_F32) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[c][k] = raw_as_f32(r.w[c][k / 4][k % 4], DT);
        } else if constexpr (DT == VQ2_DT_F16) {
            const half8_t h = __builtin_bit_cast(half8_t, r.w[c][0]);
#pragma unroll
            for (int k = 0; k < 8; k++) v[c][k] = (float)h[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[c][2 * k] = __uint_as_float(r.w[c][0][k] << 16);
                v[c][2 * k + 1] = __uint_as_float(r.w[c][0][k] & 0xFFFF0000u);
            }
        }
    }
}
template <int V, int TPR, bool VEC>
__device__ __forceinline__ void load_row(float (&v)[V][8], const void* p, int dt, int64_t row, int n, int id)
{
    if (dt == VQ2_DT_F16) {
        Raw<VQ2_DT_F16, V, VEC> r;
        load_raw<VQ2_DT_F16, V, TPR, VEC>(r, p, row, n, id);
        numbers(v, r);
    } else if (dt == VQ2_DT_BF16) {
        Raw<VQ2_DT_BF16, V, VEC> r;
        load_raw<VQ2_DT_BF16, V, TPR, VEC>(r, p, row, n, id);
        numbers(v, r);
    } else {
        Raw<VQ2_DT_F32, V, VEC> r;
        load_raw<VQ2_DT_F32, V, TPR, VEC>(r, p, row, n, id);
        numbers(v, r);
    }
}

__device__ __forceinline__ void store8(void* p, int dt, int64_t i, const float (&v)[8])
{
    if (dt == VQ2_DT_F32) {
        *(f32x4_t*)((float*)p + i) = f32x4_t{v[0], v[1], v[2], v[3]};
        *(f32x4_t*)((float*)p + i + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else if (dt == VQ2_DT_F16) {
        half8_t h;
#pragma unroll
        for (int k = 0; k < 8; k++) h[k] = (_Float16)v[k];
        *(half8_t*)((uint16_t*)p + i) = h;
    } else {
        u32x4 u;
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = bf16_pair(v[2 * k], v[2 * k + 1]);
        *(u32x4*)((uint16_t*)p + i) = u;
    }
}

// v * inv rounded to the nearest (ties to even), 8 bits each; |v * inv| <= 127
// (448) but for its rounding
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, float inv, int dt)
{
    if (dt == VQ2_DT_I8) {
        // adding 1.5 * 2^23 rounds to a whole number in the low bits
        auto q = [&](float v) { return __float_as_uint(fmaf(v, inv, 12582912.0f)); };
        const uint32_t lo = __builtin_amdgcn_perm(q(b), q(a), 0x0C0C0400u), hi = __builtin_amdgcn_perm(q(d), q(c), 0x0C0C0400u);
        return lo | hi << 16;
    }
    auto cl = [&](float v) { return v * inv != v * inv ? v * inv : fminf(fmaxf(v * inv, -448.0f), 448.0f); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(cl(a), cl(b), 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(cl(c), cl(d), r, true);
    return (uint32_t)r;
}

template <int V, int TPR, bool VEC>
__device__ __forceinline__ void store_row(const float (&v)[V][8], void* p, int dt, int64_t row, int n, int id, float inv)
{
#pragma unroll
    for (int c = 0; c < V; c++) {
        if constexpr (VEC) {
            const int i = place<V, TPR, VEC>(c, 0, id);
            if (i >= n) continue;
            if (dt <= VQ2_DT_BF16) store8(p, dt, row * n + i, v[c]);
            else
                *(u32x2*)((uint8_t*)p + row * n + i) =
                    u32x2{quant4(v[c][0], v[c][1], v[c][2], v[c][3], inv, dt), quant4(v[c][4], v[c][5], v[c][6], v[c][7], inv, dt)};
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = place<V, TPR, VEC>(c, k, id);
                if (i >= n) continue;
                if (dt <= VQ2_DT_BF16) store_from_f32(p, dt, row * n + i, v[c][k]);
                else ((uint8_t*)p)[row * n + i] = (uint8_t)quant4(v[c][k], 0.0f, 0.0f, 0.0f, inv, dt);
            }
        }
    }
}

// Rotation tables of a thread's values (VEC), two entries a word: four times
// the place the value comes from (15 bits), its sign above.  A part with an entry
// that is no place of the row gets a NaN added, which the transform spreads
// over its block, as in vq2_rht.
template <int V>
struct Tables {
    uint32_t w[V][4];
    float nan[V];
};
template <int V, int TPR>
__device__ __forceinline__ void load_tables(Tables<V>& t, const NormCall& a, int id)
{
#pragma unroll
    for (int c = 0; c < V; c++) {
        const int i = (c * TPR + id) * 8, at = i < a.n ? i : 0;
        u32x4 p[2];
        u32x2 sg = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; k++) p[k / 4][k % 4] = at + k;
        if (a.perm) {
            p[0] = *(const u32x4*)(a.perm + at);
            p[1] = *(const u32x4*)(a.perm + at + 4);
        }
        if (a.sign) sg = *(const u32x2*)(a.sign + at);
        t.nan[c] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            uint32_t q = p[k / 4][k % 4];
            if (q >= (uint32_t)a.n) {
                q = 0;
                t.nan[c] = __builtin_nanf("");
            }
            const uint32_t e = q * 4 | (sg[k / 4] >> (8 * (k % 4) + 7) & 1) << 15;
            t.w[c][k >> 1] = k & 1 ? t.w[c][k >> 1] | e << 16 : e;
        }
    }
}
template <int V>
__device__ __forceinline__ float& table_place(float* s, const Tables<V>& t, int c, int k)
{
    const uint32_t w = t.w[c][k >> 1];
    return *(float*)((char*)s + ((k & 1 ? w >> 16 : w) & 0x7FFCu));
}
template <int V>
__device__ __forceinline__ float table_sign(float v, const Tables<V>& t, int c, int k)
{
    const uint32_t w = t.w[c][k >> 1];
    return __uint_as_float(__float_as_uint(v) ^ ((k & 1 ? w : w << 16) & 0x80000000u));
}

template <int DT, int V, int TPR, bool VEC, bool ROT>
__global__ void __launch_bounds__(threads_of(TPR), 2) norm_kernel(const NormCall a, int64_t row_step)
{
    constexpr int RW = threads_of(TPR) / TPR;  // rows of a workgroup
    __shared__ __align__(16) float s_row[ROT ? V * 8 * threads_of(TPR) : 1];
    __shared__ float s_red[8];
    const int id = threadIdx.x % TPR, rw = threadIdx.x / TPR;
    float* s = s_row + (ROT ? rw * V * 8 * TPR : 0);
    // The next row's values are on their way while this one is worked on.  The
    // loads are unconditional (the last row again, x for a residual that is
    // not there): behind a branch the compiler waits for all of them at the
    // next use of any (norm_grad_kernel, 8192 rows of 6144: 200 us so).
    const void* res = a.residual ? a.residual : a.x;
    Raw<DT, V, VEC> rx, rr;
    auto fetch = [&](int64_t r0) {
        const int64_t at = min(r0 + rw, a.rows - 1);
        load_raw<DT, V, TPR, VEC>(rx, a.x, at, a.n, id);
        load_raw<DT, V, TPR, VEC>(rr, res, at, a.n, id);
    };
    fetch((int64_t)blockIdx.x * RW);
    float w[V][8];
    Tables<V> tab;
    load_row<V, TPR, VEC>(w, a.weight, a.w_dt, 0, a.n, id);
    if constexpr (ROT) load_tables<V, TPR>(tab, a, id);
    if (a.zero_centred)
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) w[c][k] += 1.0f;
    for (int64_t r0 = (int64_t)blockIdx.x * RW; r0 < a.rows; r0 += row_step) {
        const int64_t row = r0 + rw;
        const bool live = row < a.rows;
        float h[V][8];
        numbers(h, rx);
        if (a.residual) {
            float e[V][8];
            numbers(e, rr);
#pragma unroll
            for (int c = 0; c < V; c++)
#pragma unroll
                for (int k = 0; k < 8; k++) h[c][k] += e[c][k];
        }
        fetch(r0 + row_step);
        if (a.h && live) store_row<V, TPR, VEC>(h, a.h, DT, row, a.n, id, 0.0f);
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) sum[0] += h[c][k] * h[c][k];
        row_reduce<TPR>(sum, s_red, add_op);
        const float r = 1.0f / sqrtf(sum[0] / (float)a.n + a.eps);
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) h[c][k] = h[c][k] * r * w[c][k];
        if constexpr (ROT) {
            __syncthreads();  // the last row's values have been read
#pragma unroll
            for (int c = 0; c < V; c++) {
                f32x4_t* p = (f32x4_t*)(s + (c * TPR + id) * 8);
                p[0] = f32x4_t{h[c][0], h[c][1], h[c][2], h[c][3]};
                p[1] = f32x4_t{h[c][4], h[c][5], h[c][6], h[c][7]};
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < V; c++) {
#pragma unroll
                for (int k = 0; k < 8; k++) h[c][k] = table_sign(table_place(s, tab, c, k), tab, c, k);
                h[c][0] += tab.nan[c];
            }
            hadamard<V, TPR>(h, a.hb, id, s);
#pragma unroll
            for (int c = 0; c < V; c++)
#pragma unroll
                for (int k = 0; k < 8; k++) h[c][k] *= a.rht_scale;
        }
        float inv = 0.0f;
        if (a.y_dt > VQ2_DT_BF16) {
            float m[1] = {0.0f};
#pragma unroll
            for (int c = 0; c < V; c++)
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (place<V, TPR, VEC>(c, k, id) < a.n) m[0] = bits_op(m[0], fabsf(h[c][k]));
            row_reduce<TPR>(m, s_red, bits_op);
            const float top = a.y_dt == VQ2_DT_I8 ? 127.0f : 448.0f;
            // (a scale below 2^-126 would have no reciprocal)
            const bool low = m[0] > 0.0f && m[0] < top * 0x1p-126f;
            inv = low ? 0x1p126f : m[0] > 0.0f ? top / m[0] : 0.0f;
            if (live && id == 0) a.y_scale[row] = low ? 0x1p-126f : m[0] / top;
        }
        if (live) store_row<V, TPR, VEC>(h, a.y, a.y_dt, row, a.n, id, inv);
    }
}

template <int DT, int V, int TPR, bool VEC, bool ROT>
__global__ void __launch_bounds__(threads_of(TPR), 2) norm_grad_kernel(const NormCall a, int64_t row_step, float* part)
{
    constexpr int RW = threads_of(TPR) / TPR;
    __shared__ __align__(16) float s_row[ROT || RW > 1 ? V * 8 * threads_of(TPR) : 1];
    __shared__ float s_red[16];
    const int id = threadIdx.x % TPR, rw = threadIdx.x / TPR;
    float* s = s_row + (ROT ? rw * V * 8 * TPR : 0);
    const bool same = a.y_dt == DT;  // dy of h's type
    const void* gsrc = same ? a.dy : a.x;
    const void* esrc = a.dh ? a.dh : a.x;
    Raw<DT, V, VEC> rh, rg;
    auto fetch = [&](int64_t r0) {
        const int64_t at = min(r0 + rw, a.rows - 1);
        load_raw<DT, V, TPR, VEC>(rg, gsrc, at, a.n, id);
        load_raw<DT, V, TPR, VEC>(rh, a.x, at, a.n, id);
    };
    fetch((int64_t)blockIdx.x * RW);
    float w[V][8], dw[V][8];
    Tables<V> tab;
    load_row<V, TPR, VEC>(w, a.weight, a.w_dt, 0, a.n, id);
    if constexpr (ROT) load_tables<V, TPR>(tab, a, id);
#pragma unroll
    for (int c = 0; c < V; c++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (a.zero_centred) w[c][k] += 1.0f;
            dw[c][k] = 0.0f;
        }
    for (int64_t r0 = (int64_t)blockIdx.x * RW; r0 < a.rows; r0 += row_step) {
        const int64_t row = r0 + rw, at = min(row, a.rows - 1);
        const bool live = row < a.rows;
        float h[V][8], g[V][8];
        if (same) numbers(g, rg);
        else load_row<V, TPR, VEC>(g, a.dy, a.y_dt, at, a.n, id);
        numbers(h, rh);
        Raw<DT, V, VEC> re;
        load_raw<DT, V, TPR, VEC>(re, esrc, at, a.n, id);
        fetch(r0 + row_step);
        if constexpr (ROT) {
            hadamard<V, TPR>(g, a.hb, id, s);
            __syncthreads();
#pragma unroll
            for (int c = 0; c < V; c++) {
                g[c][0] += tab.nan[c];
                if ((c * TPR + id) * 8 < a.n)
#pragma unroll
                    for (int k = 0; k < 8; k++) table_place(s, tab, c, k) = table_sign(g[c][k] * a.rht_scale, tab, c, k);
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < V; c++) {
                const f32x4_t* p = (const f32x4_t*)(s + (c * TPR + id) * 8);
                const f32x4_t lo = p[0], hi = p[1];
                const bool in = (c * TPR + id) * 8 < a.n;  // (past the row nothing was written)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    g[c][k] = in ? lo[k] : 0.0f;
                    g[c][4 + k] = in ? hi[k] : 0.0f;
                }
            }
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                sum[0] += h[c][k] * h[c][k];
                sum[1] += g[c][k] * w[c][k] * h[c][k];
            }
        row_reduce<TPR>(sum, s_red, add_op);
        const float r = 1.0f / sqrtf(sum[0] / (float)a.n + a.eps), b = r * r * r * (sum[1] / (float)a.n);
        float e[V][8];
        numbers(e, re);
#pragma unroll
        for (int c = 0; c < V; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (live) dw[c][k] += g[c][k] * (h[c][k] * r);
                const float d = r * (g[c][k] * w[c][k]) - h[c][k] * b;
                e[c][k] = a.dh ? e[c][k] + d : d;
            }
        if (live) store_row<V, TPR, VEC>(e, a.y, DT, row, a.n, id, 0.0f);
    }
    if (!part) return;
    if constexpr (RW > 1) {  // the workgroup's rows, added in order
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; k++) s_row[(rw * 8 + k) * TPR + id] = dw[0][k];
        __syncthreads();
        if (rw) return;
        for (int y = 1; y < RW; y++)
#pragma unroll
            for (int k = 0; k < 8; k++) dw[0][k] += s_row[(y * 8 + k) * TPR + id];
    }
    float* o = part + (int64_t)blockIdx.x * a.n;
#pragma unroll
    for (int c = 0; c < V; c++) {
        if (VEC && place<V, TPR, VEC>(c, 0, id) < a.n) {
            store8(o, VQ2_DT_F32, place<V, TPR, VEC>(c, 0, id), dw[c]);
        } else if (!VEC) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (place<V, TPR, VEC>(c, k, id) < a.n) o[place<V, TPR, VEC>(c, k, id)] = dw[c][k];
        }
    }
}

// dw: the sums of the workgroups, 16 columns a workgroup, 64 threads a column
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* part, int chunks, int n, float* dw)
{
    __shared__ float s[64][17];
    const int x = threadIdx.x & 15, col = blockIdx.x * 16 + x, y = threadIdx.x >> 4;
    float v = 0.0f;
    if (col < n)
#pragma unroll 8
        for (int k = y; k < chunks; k += 64) v += part[(int64_t)k * n + col];
    s[y][x] = v;
    __syncthreads();
    for (int w = 32; w; w /= 2) {
        if (y < w) s[y][x] += s[y + w][x];
        __syncthreads();
    }
    if (y == 0 && col < n) dw[col] = s[0][x];
}

struct Shape {
    int v, tpr, vec, rot;
    int64_t groups;  // workgroups
};

Shape shape_of(const NormCall& c, bool grad)
{
    Shape s;
    s.rot = c.hb > 0;
    const uintptr_t ptrs = (uintptr_t)c.x | (uintptr_t)c.residual | (uintptr_t)c.weight | (uintptr_t)c.y | (uintptr_t)c.h |
                           (uintptr_t)c.dy | (uintptr_t)c.dh;
    s.vec = c.n % 8 == 0 && ptrs % 16 == 0;
    // 8 values a thread of a row where that many threads are there (a row of 1024
    // with 256 threads took twice its time), up to 32
    s.tpr = c.n <= 128 ? 16 : c.n <= 512 ? 64 : c.n <= 1024 ? 128 : c.n <= 6144 || !grad ? 256 : 512;
    s.v = (c.n + s.tpr * 8 - 1) / (s.tpr * 8);
    const int64_t per = threads_of(s.tpr) / s.tpr, rows = (c.rows + per - 1) / per;
    // forward: enough workgroups to hide each other's loads; backward: fewer,
    // each leaves a row of sums
    s.groups = std::min<int64_t>(rows, (int64_t)device_cu_count() * (grad ? (s.v <= 2 ? 4 : 2) : s.v <= 2 ? 8 : 4));
    return s;
}

template <bool GRAD, int DT, int V, int TPR>
hipError_t launch(const NormCall& c, const Shape& s, float* part)
{
    const dim3 grid((unsigned)s.groups), block(threads_of(TPR));
    const hipStream_t st = (hipStream_t)c.stream;
    const int64_t step = s.groups * (threads_of(TPR) / TPR);
    if constexpr (GRAD) {
        if (s.rot) hipLaunchKernelGGL((norm_grad_kernel<DT, V, TPR, true, true>), grid, block, 0, st, c, step, part);
        else if (s.vec) hipLaunchKernelGGL((norm_grad_kernel<DT, V, TPR, true, false>), grid, block, 0, st, c, step, part);
        else hipLaunchKernelGGL((norm_grad_kernel<DT, V, TPR, false, false>), grid, block, 0, st, c, step, part);
    } else {
        if (s.rot) hipLaunchKernelGGL((norm_kernel<DT, V, TPR, true, true>), grid, block, 0, st, c, step);
        else if (s.vec) hipLaunchKernelGGL((norm_kernel<DT, V, TPR, true, false>), grid, block, 0, st, c, step);
        else hipLaunchKernelGGL((norm_kernel<DT, V, TPR, false, false>), grid, block, 0, st, c, step);
    }
    return hipGetLastError();
}

template <bool GRAD, int DT>
hipError_t launch_shape(const NormCall& c, const Shape& s, float* part)
{
    if (s.tpr == 16) return launch<GRAD, DT, 1, 16>(c, s, part);
    if (s.tpr == 64) return launch<GRAD, DT, 1, 64>(c, s, part);
    if (s.tpr == 128) return launch<GRAD, DT, 1, 128>(c, s, part);
    if (s.v == 1) return launch<GRAD, DT, 1, 256>(c, s, part);
    if (s.tpr == 256 && s.v == 2) return launch<GRAD, DT, 2, 256>(c, s, part);
    if (s.v == 3) return launch<GRAD, DT, 3, 256>(c, s, part);
    if constexpr (GRAD) return launch<GRAD, DT, 2, 512>(c, s, part);
    else return launch<GRAD, DT, 4, 256>(c, s, part);
}

template <bool GRAD>
hipError_t launch_dt(const NormCall& c, const Shape& s, float* part)
{
    if (c.x_dt == VQ2_DT_F16) return launch_shape<GRAD, VQ2_DT_F16>(c, s, part);
    if (c.x_dt == VQ2_DT_BF16) return launch_shape<GRAD, VQ2_DT_BF16>(c, s, part);
    return launch_shape<GRAD, VQ2_DT_F32>(c, s, part);
}

}  // namespace

size_t norm_workspace_bytes(int64_t rows, int64_t n)
{
    NormCall c{};
    c.rows = rows;
    c.n = (int)n;
    const Shape s = shape_of(c, true);
    return rows == 0 ? 0 : (size_t)s.groups * n * 4;
}

int norm_launch(const NormCall& c)
{
    const Shape s = shape_of(c, false);
    const hipError_t e = launch_dt<false>(c, s, nullptr);
    return e == hipSuccess ? VQ2_OK : set_hip_error(e, "vq2_add_rms_norm");
}

int norm_grad_launch(const NormCall& c, float* dw, void* workspace)
{
    const Shape s = shape_of(c, true);
    if (c.rows) {
        const hipError_t e = launch_dt<true>(c, s, dw ? (float*)workspace : nullptr);
        if (e != hipSuccess) return set_hip_error(e, "vq2_add_rms_norm_backward");
    }
    if (!dw) return VQ2_OK;
    hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)((c.n + 15) / 16)), dim3(1024), 0, (hipStream_t)c.stream,
                       (const float*)workspace, c.rows ? (int)s.groups : 0, c.n, dw);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VQ2_OK : set_hip_error(e, "vq2_add_rms_norm_backward");
}

}  // namespace vq2
