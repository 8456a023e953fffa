// GEMM of microscaled 4-bit operands for gfx950: y[M][N] = A[M][K] . W[N][K]^T, both in
// the form of ltx_args.h, on v_mfma_scale_f32_16x16x128_f8f6f4: a lane's operand is a
// group of 32 codes (16 bytes) and its scale, which the instruction applies, so nothing
// is unpacked. f32 accumulation.
//
// Workgroup: 4 waves in a 2 x 2 grid, output tile 32 NI x 32 NI, a wave NI x NI blocks of
// 16 x 16. Bytes lie as in the four-wave 16-bit GEMM, 128 of them being 256 k: K goes in
// tiles of 256 through LDS by LDS DMA in two stages, rows of 128 B with 16-byte chunk c of
// row r in slot c ^ ((r >> 1) & 7), a tile is two steps of 128 k, and in step s lanes
// 16 h .. 16 h + 15 read chunk 4 s + h of their rows: groups 4 s + h. Scale words come the
// same way, 64 rows an instruction (wave w: matrix w / 2, step w % 2); a lane reads its
// group's byte.
//
// Schedule as there: one barrier per K-tile at the middle of the pair of steps that
// straddles two tiles; after the barrier behind tile k's step 0 the DMA of tile k + 2 goes
// to the stage that tile k came from, while tile k's step 1 and tile k + 1's step 0 are
// multiplied, each beside the fragment reads of the next.
//
// The tiles of a row go to an even count. Codes behind the last group are those of the next
// row (or zeros behind the last), which are numbers whatever they are; their scale words lie
// behind the resource's end and read as zeros, 2^-127 on both sides, and what such products
// add is below f32's smallest number.
#pragma once
#include "gemm_common.h"
#include "ltx_fp4.h"

typedef __attribute__((address_space(3))) void* lds_vptr;
typedef int i32x8 __attribute__((ext_vector_type(8)));

#define MX4_RSRC_W3 0x00020000
#define MX4_WAIT_VM0 ((7 << 4) | (15 << 8))
#define MX4_WAIT_ALL0 (7 << 4)

// One __shared__ object per matrix and stage: the compiler's LDS-DMA alias tracking then
// waits only for the stage that a read touches. KIND 0: A, 1: W, 2: scale words [A step 0,
// A step 1, W step 0, W step 1][rows].
template <int KIND, int S, int BYTES>
__device__ __forceinline__ uint8_t* mx4_stage() {
    __shared__ __attribute__((aligned(1024))) uint8_t buf[BYTES];
    return buf;
}

// Offsets through an empty volatile asm at the point of use, so that the LDS addresses
// derived from them are not kept as a register each.
__device__ __forceinline__ uint32_t mx4_vofs(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int mx4_sofs(int x) {
    asm volatile("" : "+s"(x));
    return x;
}

__device__ __forceinline__ f32x4 mx4_mfma(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
    const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

template <typename T, int NI>
struct Mx4Gemm {
    static constexpr int TM = 32 * NI;       // rows and columns of the output tile
    static constexpr int NR = 2 * NI;        // fragment reads of a step, code DMA instructions of a K-tile
    static constexpr int NS = NI / 2;        // scale DMA instructions of a K-tile and wave
    const LtxMx4LinearArgs& a;
    f32x4 acc[NI][NI];
    __amdgpu_buffer_rsrc_t ra_, rb_, rs_;
    uint32_t ga[NI], gb[NI];    // per-lane source offsets of the DMA instructions, K-tile 0
    uint32_t gs, gstep;         // of the scale words, and bytes to the next step's
    int lw, lsw;                // this wave's DMA destinations within a stage (codes, scale words)
    uint32_t offa[2], offb[2];  // fragment reads of step s (row block i adds 2048 i)
    uint32_t sa_, sb_;          // and of the scale bytes, step 0 (row block i adds 64 i)
    u32x4 fa0[NI], fb0[NI], fa1[NI], fb1[NI];
    uint32_t xa0[NI], xb0[NI], xa1[NI], xb1[NI];

    __device__ __forceinline__ Mx4Gemm(const LtxMx4LinearArgs& args) : a(args) {}

    template <int S>
    static __device__ __forceinline__ uint8_t* stage_a() {
        return mx4_stage<0, S, 128 * TM>();
    }
    template <int S>
    static __device__ __forceinline__ uint8_t* stage_b() {
        return mx4_stage<1, S, 128 * TM>();
    }
    template <int S>
    static __device__ __forceinline__ uint8_t* stage_s() {
        return mx4_stage<2, S, 16 * TM>();
    }

    // slot i of the reads of step STEP of stage S, in the order the MFMAs need them:
    // A0, W0 .. , A1 .. , each with its scale
    template <int S, int STEP>
    __device__ __forceinline__ void read1(int g, u32x4 (&ya)[NI], u32x4 (&yb)[NI], uint32_t (&za)[NI],
                                          uint32_t (&zb)[NI], const uint8_t* sa, const uint8_t* sb, const uint8_t* pa,
                                          const uint8_t* pb) {
        if (g == 0 || g > NI) {
            const int i = g == 0 ? 0 : g - NI;
            za[i] = pa[64 * i];
            ya[i] = *(const u32x4*)(sa + 2048 * i);
        } else {
            zb[g - 1] = pb[64 * (g - 1)];
            yb[g - 1] = *(const u32x4*)(sb + 2048 * (g - 1));
        }
    }
    template <int S, int STEP>
    __device__ __forceinline__ void read_all(u32x4 (&ya)[NI], u32x4 (&yb)[NI], uint32_t (&za)[NI], uint32_t (&zb)[NI]) {
        const uint8_t* sa = stage_a<S>() + mx4_vofs(offa[STEP]);
        const uint8_t* sb = stage_b<S>() + mx4_vofs(offb[STEP]);
        const uint8_t* pa = stage_s<S>() + mx4_vofs(sa_) + 4 * TM * STEP;
        const uint8_t* pb = stage_s<S>() + mx4_vofs(sb_) + 4 * TM * STEP;
#pragma unroll
        for (int g = 0; g < NR; g++) read1<S, STEP>(g, ya, yb, za, zb, sa, sb, pa, pb);
    }

    // DMA instruction g of K-tile k into stage S: scale words first, then A, then W. The
    // whole offset is the lane's, so that the bounds check covers it.
    template <int S>
    __device__ __forceinline__ void dma1(int g, int k, uint8_t* da, uint8_t* db, uint8_t* ds) {
        if (g < NS)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_, (lds_vptr)(ds + 256 * g), 4, gs + 256 * g + 2 * k * gstep, 0, 0,
                                                     0);
        else if (g < NS + NI)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra_, (lds_vptr)(da + 1024 * (g - NS)), 16, ga[g - NS] + 128 * k, 0,
                                                     0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb_, (lds_vptr)(db + 1024 * (g - NS - NI)), 16,
                                                     gb[g - NS - NI] + 128 * k, 0, 0, 0);
    }
    template <int S>
    __device__ __forceinline__ void dma(int k) {
        const int l = mx4_sofs(lw), ls = mx4_sofs(lsw);
#pragma unroll
        for (int g = 0; g < NS + NR; g++) dma1<S>(g, k, stage_a<S>() + l, stage_b<S>() + l, stage_s<S>() + ls);
    }

    __device__ __forceinline__ void mfma_all(const u32x4 (&xa)[NI], const u32x4 (&xb)[NI], const uint32_t (&sa)[NI],
                                             const uint32_t (&sb)[NI]) {
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < NI; j++) acc[i][j] = mx4_mfma(xa[i], xb[j], acc[i][j], sa[i], sb[j]);
    }

    // The MFMAs of one step with the reads of another (stage RS, step RSTEP) and, when DMA,
    // the DMA instructions of tile kd into stage DS, spread evenly between them.
    template <int RS, int RSTEP, int DS, bool DMA>
    __device__ __forceinline__ void region(const u32x4 (&xa)[NI], const u32x4 (&xb)[NI], const uint32_t (&sa)[NI],
                                           const uint32_t (&sb)[NI], u32x4 (&ya)[NI], u32x4 (&yb)[NI],
                                           uint32_t (&za)[NI], uint32_t (&zb)[NI], int kd) {
        const uint8_t* pa = stage_a<RS>() + mx4_vofs(offa[RSTEP]);
        const uint8_t* pb = stage_b<RS>() + mx4_vofs(offb[RSTEP]);
        const uint8_t* qa = stage_s<RS>() + mx4_vofs(sa_) + 4 * TM * RSTEP;
        const uint8_t* qb = stage_s<RS>() + mx4_vofs(sb_) + 4 * TM * RSTEP;
        const int l = DMA ? mx4_sofs(lw) : 0, ls = DMA ? mx4_sofs(lsw) : 0;
        constexpr int ND = NS + NR;
        int rd = 0, dd = 0;
#pragma unroll
        for (int m = 0; m < NI * NI; m++) {
            acc[m / NI][m % NI] = mx4_mfma(xa[m / NI], xb[m % NI], acc[m / NI][m % NI], sa[m / NI], sb[m % NI]);
            const int r1 = (m + 1) * NR / (NI * NI), d1 = DMA ? (m + 1) * ND / (NI * NI) : 0;
            if (r1 > rd || d1 > dd) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (; rd < r1; rd++) read1<RS, RSTEP>(rd, ya, yb, za, zb, pa, pb, qa, qb);
#pragma unroll
                for (; dd < d1; dd++) dma1<DS>(dd, kd, stage_a<DS>() + l, stage_b<DS>() + l, stage_s<DS>() + ls);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    __device__ __forceinline__ void meet() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(MX4_WAIT_ALL0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }

    // Entered after a barrier: tile k in stage S with its step-1 fragments in registers,
    // tile k + 1 landed in stage S ^ 1, stage S read by every wave.
    template <int S, bool DMA>
    __device__ __forceinline__ void pair(int k) {
        region<S ^ 1, 0, S, DMA>(fa1, fb1, xa1, xb1, fa0, fb0, xa0, xb0, k + 2);
        __builtin_amdgcn_sched_barrier(0);
        region<S ^ 1, 1, S, false>(fa0, fb0, xa0, xb0, fa1, fb1, xa1, xb1, 0);
        meet();
    }

    // 32 rows at a time through a private patch, so that rows of y leave in 16-byte pieces
    __device__ __forceinline__ void store(float* patch, int mw, int nw) {
        constexpr int WN = 16 * NI, LD = WN + 4;
        const int lane = opaque_tid() & 63;
        const bool f32 = a.out_f32 != 0;
        const int per = f32 ? 4 : 8, lanes = WN / per, step = 64 / lanes;
        const int c = per * (lane % lanes), r0 = lane / lanes, n = nw + c;
        float bias[8];
#pragma unroll
        for (int e = 0; e < 8; e++) bias[e] = a.bias && e < per && n + e < a.N ? a.bias[n + e] : 0.f;
#pragma unroll
        for (int b = 0; b < NI / 2; b++) {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < NI; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        patch[(16 * e + 4 * (lane >> 4) + r) * LD + 16 * j + (lane & 15)] = acc[2 * b + e][j][r];
            for (int r = r0; r < 32; r += step) {
                const int m = mw + 32 * b + r;
                if (m >= a.M || n >= a.N) continue;
                float v[8];
                *(f32x4*)v = *(const f32x4*)(patch + r * LD + c);
                *(f32x4*)(v + 4) = f32 ? f32x4{0, 0, 0, 0} : *(const f32x4*)(patch + r * LD + c + 4);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[e] += bias[e];
                    if (a.gelu) v[e] = gelu_tanh(v[e]);
                }
                const size_t at = (size_t)m * a.N + n;
                if (f32) {
                    float* y = (float*)a.y + at;
                    if (a.wide && n + 4 <= a.N)
                        *(f32x4*)y = f32x4{v[0], v[1], v[2], v[3]};
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n + e < a.N) y[e] = v[e];
                } else {
                    uint16_t* y = (uint16_t*)a.y + at;
                    if (a.wide && n + 8 <= a.N)
                        *(u32x4*)y = u32x4{Op<T>::cvt2(v[0], v[1]), Op<T>::cvt2(v[2], v[3]), Op<T>::cvt2(v[4], v[5]),
                                           Op<T>::cvt2(v[6], v[7])};
                    else
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (n + e < a.N) y[e] = Op<T>::bits(v[e]);
                }
            }
        }
    }

    __device__ __forceinline__ void run() {
        const int tid = threadIdx.x, lane = tid & 63;
        const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = 16 * NI * (w >> 1), wn = 16 * NI * (w & 1);
        const int G = a.K / 128, nk = 2 * ((G + 3) / 4);
        const uint32_t row = (uint32_t)a.K / 2;
        lw = 1024 * NI * w;
        lsw = 4 * TM * w;
        {
            const int h = lane >> 4, r = lane & 15;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                offa[s] = (wm + r) * 128 + 16 * ((4 * s + h) ^ ((r >> 1) & 7));
                offb[s] = (wn + r) * 128 + 16 * ((4 * s + h) ^ ((r >> 1) & 7));
            }
            sa_ = 4 * (wm + r) + h;
            sb_ = 8 * TM + 4 * (wn + r) + h;
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int tr = 8 * (NI * w + i) + (lane >> 3);
            ga[i] = gb[i] = (uint32_t)tr * row + 16u * ((lane & 7) ^ ((tr >> 1) & 7));
        }
        uint8_t* patch = w == 0 ? stage_a<0>() : w == 1 ? stage_a<1>() : w == 2 ? stage_b<0>() : stage_b<1>();
        const int ntiles = a.tiles_m * a.tiles_n;
        for (int item = blockIdx.x; item < ntiles; item += gridDim.x) {
            const TileIdx ti = tile_of(item, a.tiles_m, a.tiles_n);
            const int m0 = ti.tm * TM, n0 = ti.tn * TM;
            // resources that begin at the tile's first row: rows behind the last read as zeros
            ra_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.a + (size_t)m0 * row), 0,
                                                    (int)((uint32_t)min(TM, a.M - m0) * row), MX4_RSRC_W3);
            rb_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (size_t)n0 * row), 0,
                                                    (int)((uint32_t)min(TM, a.N - n0) * row), MX4_RSRC_W3);
            const int rows = w < 2 ? a.M : a.N, first = w < 2 ? m0 : n0;
            rs_ = __builtin_amdgcn_make_buffer_rsrc((void*)((w < 2 ? a.as : a.ws) + 4 * (size_t)first), 0,
                                                    (int)(4u * ((uint32_t)G * (uint32_t)rows - (uint32_t)first)),
                                                    MX4_RSRC_W3);
            gstep = 4u * (uint32_t)rows;
            gs = 4 * lane + (w & 1) * gstep;
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int j = 0; j < NI; j++) acc[i][j] = f32x4{0, 0, 0, 0};
            dma<0>(0);
            __builtin_amdgcn_s_waitcnt(MX4_WAIT_VM0);
            __builtin_amdgcn_s_barrier();
            dma<1>(1);
            read_all<0, 0>(fa0, fb0, xa0, xb0);
            read_all<0, 1>(fa1, fb1, xa1, xb1);
            mfma_all(fa0, fb0, xa0, xb0);  // tile 0, step 0
            meet();
            for (int k = 0; k < nk - 2; k += 2) {
                pair<0, true>(k);
                pair<1, true>(k + 1);
            }
            pair<0, false>(nk - 2);
            mfma_all(fa1, fb1, xa1, xb1);  // tile nk - 1, step 1
            meet();
            // every wave has passed the last barrier: the stages are free
            store((float*)patch, m0 + wm, n0 + wn);
            meet();
        }
    }
};

#define MX4_GEMM_KERNEL(NAME, T_, NI_, PER_)                                               \
    extern "C" __global__ void __launch_bounds__(256, PER_) NAME(const LtxMx4LinearArgs a) { \
        Mx4Gemm<T_, NI_> k(a);                                                             \
        k.run();                                                                           \
    }
