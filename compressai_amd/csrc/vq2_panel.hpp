// vq2_panel.hpp -- operands of a product in the order the matrix cores read
// them ("panels"), and the product of two panels.
//
// A panel holds rows of k values as blocks of 16 rows x 32 values, 1 KiB
// each, the blocks of a 16-row tile one after the other: lane l of a wave
// finds row l % 16, values 8 (l / 16) .. + 7 at its own 16 bytes, which is
// one operand of v_mfma_f32_16x16x32_f16.  Loads into LDS and reads from it
// are whole contiguous KiB, without bank conflicts and without index
// arithmetic, and whoever writes a panel chooses the order of rows and
// values freely as long as its partner panel has the same order of values.
#pragma once

#include "vq2_common.hpp"

namespace vq2 {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

struct Eight {
    float v[8];
};

// 8 elements from a 16-byte (8-byte for 8-bit types) aligned address
__device__ __forceinline__ Eight load8(const void* p, int dt, int64_t i)
{
    Eight r;
    if (dt == VQ2_DT_F32) {
        const f32x4_t a = *(const f32x4_t*)((const float*)p + i), b = *(const f32x4_t*)((const float*)p + i + 4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            r.v[k] = a[k];
            r.v[4 + k] = b[k];
        }
    } else if (dt == VQ2_DT_F16) {
        const half8_t h = *(const half8_t*)((const uint16_t*)p + i);
#pragma unroll
        for (int k = 0; k < 8; k++) r.v[k] = (float)h[k];
    } else if (dt == VQ2_DT_BF16) {
        const u32x4 u = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            r.v[2 * k] = __uint_as_float(u[k] << 16);
            r.v[2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u);
        }
    } else {
        const u32x2 u = *(const u32x2*)((const uint8_t*)p + i);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if (dt == VQ2_DT_I8) {
#pragma unroll
                for (int j = 0; j < 4; j++) r.v[4 * k + j] = (float)((int)(u[k] << (24 - 8 * j)) >> 24);
            } else {
                r.v[4 * k] = __builtin_amdgcn_cvt_f32_fp8((int)u[k], 0);
                r.v[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8((int)u[k], 1);
                r.v[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8((int)u[k], 2);
                r.v[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8((int)u[k], 3);
            }
        }
    }
    return r;
}

// two values rounded to bf16, one instruction
__device__ __forceinline__ uint32_t bf16_pair(float a, float b)
{
    typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf2_t{(__bf16)a, (__bf16)b});
}

// 1 KiB of a panel straight into LDS (no registers); l is wave-uniform, the
// lanes' 16 bytes land in order behind it.
__device__ __forceinline__ void panel_to_lds(const half8_t* g, half8_t* l)
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// Product of a workgroup of 2 x 2 waves: wave tiles of 16 MT rows of panel a
// (weights) times 64 rows of panel b (tokens).  Bound by the matrix cores and
// the epilogues between their products (busy in 59 to 78 % of the cycles), on long runs
// with lower clocks: 32768 x 4096 x 2048 takes 440 to 460 us with the loss's statistics
// behind it (1.25 to 1.19 PFLOP/s), 12288 x 4096 x 2048 183 to 196 with the gated block's
// (1.13 to 1.05).  A k tile is 12 KiB of LDS reads for 32 matrix
// instructions of a wave (MT 8): larger tiles leave no registers for an epilogue.
constexpr int PG_WM = 2, PG_WN = 2, PG_NT = 4, PG_BUF = 3;
constexpr int PG_THREADS = 64 * PG_WM * PG_WN;
constexpr int PG_N = 16 * PG_WN * PG_NT;  // tokens of a workgroup
constexpr int pg_m(int MT) { return 16 * PG_WM * MT; }
// PG_BUF stages of one k tile in LDS (with 8 stages and a workgroup a CU, short
// products were no faster)
constexpr int pg_lds(int MT) { return (PG_WM * MT + PG_WN * PG_NT) * PG_BUF * 1024; }

struct PanelGemmArgs {
    const half8_t* a;  // [gm * PG_WM * MT][a_kt][64]
    const half8_t* b;  // [gn * PG_WN * PG_NT][b_kt][64]
    int a_kt, b_kt;    // k tiles; a_kt is b_kt, or twice that: b is read again for the second part of a
    int gm, gn, gz;    // workgroup tiles, and slices of the k tiles
};

// The workgroup's place: XCD x (blockIdx % 8) takes a contiguous share of the
// tiles, walked in groups of 4 tiles of a by all tiles of b, so the 64
// workgroups of an XCD share 4 + 16 panel tiles in its L2.
__device__ __forceinline__ void panel_tile(const PanelGemmArgs& g, int& bm, int& bn, int& bz)
{
    constexpr int GW = 4;
    const int nb = gridDim.x, x = blockIdx.x % 8, per = nb / 8, rem = nb % 8;
    int id = x * per + min(x, rem) + blockIdx.x / 8;
    bz = id / (g.gm * g.gn);
    id -= bz * g.gm * g.gn;
    const int grp = id / (GW * g.gn), in = id - grp * GW * g.gn, w = min(GW, g.gm - grp * GW);
    bm = grp * GW + in % w;
    bn = in / w;
}

// acc[i][j][e]: row 16 (first tile of a + i) + 4 (lane / 16) + e of a, row
// 16 (first tile of b + j) + lane % 16 of b.
template <int MT>
__device__ __forceinline__ void panel_product(const PanelGemmArgs& g, int bm, int bn, int bz, f32x4_t (&acc)[MT][PG_NT])
{
    extern __shared__ __align__(16) half8_t s_panel[];
    constexpr int TA = PG_WM * MT, TB = PG_WN * PG_NT, ST = TA + TB, W = PG_WM * PG_WN, L = ST / W;
    static_assert(ST % W == 0, "the waves load the same number of blocks");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % PG_WM, wn = wave / PG_WM;
    const int k0 = (int)((int64_t)g.a_kt * bz / g.gz), nst = (int)((int64_t)g.a_kt * (bz + 1) / g.gz) - k0;
    // this wave loads the blocks wave * L .. + L - 1 of every stage
    const half8_t* src[L];
#pragma unroll
    for (int i = 0; i < L; i++) {
        const int f = wave * L + i;
        src[i] = (f < TA ? g.a + (int64_t)(bm * TA + f) * g.a_kt * 64 : g.b + (int64_t)(bn * TB + f - TA) * g.b_kt * 64) + lane;
    }
    int slot = 0;
    auto load = [&](int stage) {
        const int k = k0 + min(stage, nst - 1);  // past the end: again the last, read by nobody
        const int kb = k >= g.b_kt ? k - g.b_kt : k;
        half8_t* d = s_panel + (slot * ST + wave * L) * 64;
        slot = slot + 1 == PG_BUF ? 0 : slot + 1;
#pragma unroll
        for (int i = 0; i < L; i++) panel_to_lds(src[i] + (int64_t)(wave * L + i < TA ? k : kb) * 64, d + i * 64);
    };
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < PG_NT; j++) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < PG_BUF - 1; i++) load(i);
    int rd = 0;
    for (int st = 0; st < nst; st++) {
        // all but the newest stage of this wave's loads have landed, and with
        // the barrier every wave's; the same barrier says that every wave has
        // read the buffer that the next load overwrites
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(L * (PG_BUF - 2)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const half8_t* s = s_panel + rd * ST * 64 + lane;
        rd = rd + 1 == PG_BUF ? 0 : rd + 1;
        half8_t fa[MT], fb[PG_NT];
#pragma unroll
        for (int j = 0; j < PG_NT; j++) fb[j] = s[(TA + wn * PG_NT + j) * 64];
#pragma unroll
        for (int i = 0; i < MT; i++) fa[i] = s[(wm * MT + i) * 64];
        load(st + PG_BUF - 1);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < PG_NT; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
    }
    // nothing may still be on its way to LDS when the workgroup ends
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace vq2
