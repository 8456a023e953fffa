// GEMM of microscaled 4-bit operands for gfx950: y[M][N] = A[M][K] . W[N][K]^T, both in
// the form of ltx_args.h, on v_mfma_scale_f32_32x32x64_f8f6f4: a lane's operand is a group
// of 32 codes (16 bytes) and its scale, which the instruction applies, so nothing is
// unpacked. f32 accumulation. (From registers and on random operands 32 x 32 x 64 runs at
// 6.4 PFLOP/s, 16 x 16 x 128 at 7.2; with an LDS read for every two products 5.7 and 5.5, twice
// the reads a flop in the latter: csrc/tools/mfma_ceiling.hip.)
//
// Workgroup: 4 waves in a 2 x 2 grid, output tile 64 NB x 64 NB, a wave NB x NB blocks of
// 32 x 32. K goes in tiles of 256 (128 bytes of a row) through LDS by LDS DMA in two stages,
// 16-byte chunk c of row r in slot c ^ ((r >> 1) & 7): 16 consecutive rows of one chunk cover
// the 64 banks once. A tile is four steps of 64 k; in step t lanes 32 h .. 32 h + 31 read
// chunk 2 t + h, a group, of their rows. Scale words come the same way, 64 rows an
// instruction (wave w: matrix w / 2, groups 4 (w % 2) .. + 3 of the tile); a lane takes a
// word for two steps and moves its two bytes to where the instruction's selector finds them.
//
// Schedule: one barrier a tile, between its steps 2 and 3. There each wave has the
// fragments of step 3 in registers, so the stage is free, and its DMA of the next tile has
// landed. Behind it the DMA of the tile after next goes out, beside the products of steps 3
// and 0, each step's beside the fragment reads of the next.
//
// The tiles of a row go to an even count. Codes behind the last group are those of the next
// row (or zeros behind the last), which are numbers whatever they are; their scale words lie
// behind the resource's end and read as zeros, 2^-127 on both sides, and what such products
// add is below f32's smallest number.
//
// Bound: 28,672 x 4,096 x 16,384 (f32 out) 830 us, 4.63 PFLOP/s, where the instruction with
// its LDS reads comes to 5.7; the K loop alone runs at about 5.0 (an operand byte is read
// from LDS once a wave and row or column block), and a 256 x 256 tile costs about 5 us beside
// it, y's stores, which the next tile's operands overlap. 2,048 x 12,288 x 4,096 is 1.5
// rounds of tiles: 61 us, 3.4 PFLOP/s.
#pragma once
#include "gemm_common.h"
#include "ltx_fp4.h"

typedef __attribute__((address_space(3))) void* lds_vptr;
typedef int i32x8 __attribute__((ext_vector_type(8)));

#define MX4_RSRC_W3 0x00020000
// s_waitcnt: vmcnt(n) and lgkmcnt(0)
#define MX4_WAIT(n) (((n) & 15) | (((n) >> 4) << 14) | (7 << 4))
#define MX4_WAIT_LGKM0 (15 | (3 << 14) | (7 << 4))

// One __shared__ object per matrix and stage: the compiler's LDS-DMA alias tracking then
// waits only for the stage that a read touches. KIND 0: A, 1: W, 2: scale words [A groups 0
// .. 3, A 4 .. 7, W 0 .. 3, W 4 .. 7][rows].
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

__device__ __forceinline__ i32x8 mx4_operand(u32x4 a) {
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
}
__device__ __forceinline__ f32x4 mx4_mfma16(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(a), mx4_operand(b), c, 4, 4, 0, (int)sa, 0,
                                                            (int)sb);
}
// B: the byte of both scale words that counts
template <int B>
__device__ __forceinline__ f32x16 mx4_mfma32(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(a), mx4_operand(b), c, 4, 4, B, (int)sa, B,
                                                           (int)sb);
}

// Out: the type of y, f32 or 16-bit. WIDE: its rows start on 16 bytes. KG: groups of four
// waves that take a tile's K-tiles in turn, each with stages of its own, and whose sums are
// added in the groups' order: where there are few tiles, a K-tile's latency is what counts
// (64 x 64 tiles, K = 16,384: 0.5 us a K-tile, of which 0.05 are products).
template <typename Out, int NB, bool GELU, bool WIDE, int KG>
struct Mx4Gemm {
    static constexpr int TM = 64 * NB;       // rows and columns of the output tile
    static constexpr int ND = 2 * NB;        // code DMA instructions of a K-tile, wave and matrix
    static constexpr int NS = NB;            // scale DMA instructions of a K-tile and wave
    static constexpr int NI = NS + 2 * ND;   // DMA instructions of a K-tile and wave
    const LtxMx4LinearArgs& a;
    f32x16 acc[NB][NB];
    __amdgpu_buffer_rsrc_t ra_, rb_, rs_;
    uint32_t ga[2];             // per-lane source offsets of even and odd DMA instructions, K-tile 0
    uint32_t gs, gstep;         // of the scale words, and bytes to those of the next 128 k
    int lw, lsw;                // this wave's DMA destinations within a stage (codes, scale words)
    uint32_t off, soff;         // A's fragments of step 0 (row block i adds 4096 i) and scale words (128 i)
    int ofw, sofw;              // from there to W's
    uint32_t shift;
    int kg;                     // this wave's group
    u32x4 fa[2][NB], fb[2][NB];     // fragments of even and odd steps
    uint32_t xa[2][NB], xb[2][NB];  // scale words of the tile's first and last two steps

    __device__ __forceinline__ Mx4Gemm(const LtxMx4LinearArgs& args) : a(args) {}

    template <int S>
    static __device__ __forceinline__ uint8_t* stage_a() {
        return mx4_stage<0, S, 128 * TM * KG>();
    }
    template <int S>
    static __device__ __forceinline__ uint8_t* stage_b() {
        return mx4_stage<1, S, 128 * TM * KG>();
    }
    template <int S>
    static __device__ __forceinline__ uint8_t* stage_s() {
        return mx4_stage<2, S, 16 * TM * KG>();
    }

    // DMA instruction g of K-tile k into stage S: scale words first, then A, then W. (The
    // bounds check takes the scalar offset in.)
    template <int S>
    __device__ __forceinline__ void dma1(int g, int k, int l, int ls) {
        if (g < NS)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_, (lds_vptr)(stage_s<S>() + ls + 256 * g), 4,
                                                     gs, 2 * (KG * k + kg) * gstep + 256 * g, 0, 0);
        else if (g < NS + ND)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra_, (lds_vptr)(stage_a<S>() + l + 1024 * (g - NS)), 16,
                                                     ga[(g - NS) & 1],
                                                     128 * (KG * k + kg) + 16 * a.K * ((g - NS) >> 1 << 1) / 4, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb_, (lds_vptr)(stage_b<S>() + l + 1024 * (g - NS - ND)), 16,
                                                     ga[(g - NS) & 1],
                                                     128 * (KG * k + kg) + 16 * a.K * ((g - NS - ND) >> 1 << 1) / 4, 0, 0);
    }
    template <int S>
    __device__ __forceinline__ void dma(int k) {
        const int l = mx4_sofs(lw), ls = mx4_sofs(lsw);
#pragma unroll
        for (int g = 0; g < NI; g++) dma1<S>(g, k, l, ls);
    }

    // read g of a step, in the order the products need them (A0, W0 .., A1 ..); even steps
    // bring the scale words of two
    template <int STEP>
    __device__ __forceinline__ void read1(int g, const uint8_t* pa, const uint8_t* pb, const uint8_t* qa,
                                          const uint8_t* qb) {
        constexpr int F = STEP & 1, X = STEP >> 1;
        if (g == 0 || g > NB) {
            const int i = g == 0 ? 0 : g - NB;
            if (F == 0) xa[X][i] = *(const uint32_t*)(qa + 128 * i);
            fa[F][i] = *(const u32x4*)(pa + 4096 * i);
        } else {
            if (F == 0) xb[X][g - 1] = *(const uint32_t*)(qb + 128 * (g - 1));
            fb[F][g - 1] = *(const u32x4*)(pb + 4096 * (g - 1));
        }
    }

    // The products of step STEP (4: none; FIRST: the tile's first, onto zero) with the reads of
    // step RSTEP of stage RS (4: none) and the DMA instructions g0 .. g1 - 1 of tile kd into
    // stage DS, spread evenly between them.
    template <int STEP, int RS, int RSTEP, int DS, bool FIRST = false>
    __device__ __forceinline__ void region(int g0, int g1, int kd) {
        constexpr int F = STEP & 1, X = (STEP >> 1) & 1, NM = NB * NB, NR = RSTEP < 4 ? 2 * NB : 0, R = RSTEP & 3;
        // (chunk 2 t + h in its slot: the bits of 2 t flip)
        const uint32_t at = mx4_vofs(off) ^ (32 * R), sat = mx4_vofs(soff);
        const uint8_t* pa = stage_a<RS>() + at;
        const uint8_t* pb = stage_b<RS>() + at + mx4_sofs(ofw);
        const uint8_t* qa = stage_s<RS>() + sat + 4 * TM * (R >> 1);
        const uint8_t* qb = stage_s<RS>() + sat + mx4_sofs(sofw) + 4 * TM * (R >> 1);
        const int l = mx4_sofs(lw), ls = mx4_sofs(lsw);
        if (STEP < 4 && F == 0) {  // the lane's bytes: 0 for this step, 2 for the next
#pragma unroll
            for (int i = 0; i < NB; i++) {
                xa[X][i] >>= shift;
                xb[X][i] >>= shift;
            }
        }
        int rd = 0, dd = g0;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const int i = m / NB, j = m % NB;
            if (STEP < 4)
                acc[i][j] = mx4_mfma32<2 * F>(fb[F][j], fa[F][i], FIRST ? f32x16{0} : acc[i][j], xb[X][j], xa[X][i]);
            const int r1 = (m + 1) * NR / NM, d1 = g0 + (m + 1) * (g1 - g0) / NM;
            if (r1 > rd || d1 > dd) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (; rd < r1; rd++) read1<R>(rd, pa, pb, qa, qb);
#pragma unroll
                for (; dd < d1; dd++) dma1<DS>(dd, kd, l, ls);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // WAIT: also for the DMA (and stores) under way
    template <bool WAIT = true>
    __device__ __forceinline__ void meet() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(WAIT ? MX4_WAIT(0) : MX4_WAIT_LGKM0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }

    // The products stay ahead of this: the compiler moved those of the last steps behind the
    // epilogue's branches, away from the reads they run beside.
    __device__ __forceinline__ void hold() {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++) {
                if constexpr (NB == 4)
                    asm volatile("" : "+a"(acc[i][j]));
                else
                    asm volatile("" : "+v"(acc[i][j]));
            }
    }

    // Tile k of stage S, from behind its step 2: entered after a barrier, the fragments of
    // its step 3 in registers and tile k + 1 in stage S ^ 1. To the same point of tile k + 1.
    template <int S, bool DMA>
    __device__ __forceinline__ void tile(int k) {
        constexpr int half = DMA ? (NI + 1) / 2 : 0, all = DMA ? NI : 0;
        region<3, S ^ 1, 0, S>(0, half, k + 2);
        region<0, S ^ 1, 1, S>(half, all, k + 2);
        region<1, S ^ 1, 2, S>(0, 0, 0);
        region<2, S ^ 1, 3, S>(0, 0, 0);
        meet();
    }

    // The groups' sums into the first one's, through the stages, which are free; true there.
    __device__ __forceinline__ bool sum_groups(int w) {
        const int lane = threadIdx.x & 63;
        auto place = [&](int g, int b) {  // 16 KB a block of a group
            constexpr int each = TM * KG / 128;
            const int s = (g - 1) * NB * NB + b;
            uint8_t* at = s / each == 0 ? stage_a<0>() : s / each == 1 ? stage_a<1>() : s / each == 2 ? stage_b<0>() : stage_b<1>();
            return (f32x4*)(at + 16384 * (s % each) + 4096 * w) + lane;
        };
#pragma unroll
        for (int g = 1; g < KG; g++) {
            if (kg != g) continue;
#pragma unroll
            for (int b = 0; b < NB * NB; b++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f32x16& x = acc[b / NB][b % NB];
                    place(g, b)[64 * q] = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                }
        }
        __syncthreads();
        if (kg > 0) return false;
#pragma unroll
        for (int g = 1; g < KG; g++)
#pragma unroll
            for (int b = 0; b < NB * NB; b++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f32x4 x = place(g, b)[64 * q];
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[b / NB][b % NB][4 * q + e] += x[e];
                }
        return true;
    }

    // y of the wave's blocks, through a resource that begins at the tile's first row: rows
    // behind the last, and columns (offset ~0), are not stored, without a branch. W's rows are
    // the products' rows, so that a lane holds runs of four columns of one row of y; in 16 bits
    // the lanes' halves exchange two runs, and each stores eight columns. Nothing goes through
    // LDS, whose stages hold the next tile's operands.
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t ry, int wm, int nw) {
        const int lane = opaque_tid() & 63, h = lane >> 5;
        constexpr int E = sizeof(Out);
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int n = nw + 32 * j + 4 * h;
            f32x4 bias[4];
#pragma unroll
            for (int g = 0; g < 4; g++) bias[g] = f32x4{0, 0, 0, 0};
            if (a.bias && nw + 32 * (j + 1) <= a.N) {
                // scalar loads: a vector load's wait would be for the DMA ahead of it too
                typedef const __attribute__((address_space(4))) float* scalar_ptr;
                const scalar_ptr b = (scalar_ptr)(uintptr_t)(a.bias + nw + 32 * j);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int c = 8 * (r >> 2) + (r & 3);
                    const float lo = b[c], hi = b[c + 4];
                    bias[r >> 2][r & 3] = h ? hi : lo;
                }
            } else if (a.bias && nw + 32 * j < a.N) {
                const __amdgpu_buffer_rsrc_t rb =
                    __builtin_amdgcn_make_buffer_rsrc((void*)(a.bias + nw), 0, 4 * (a.N - nw), MX4_RSRC_W3);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    bias[r >> 2][r & 3] = __builtin_bit_cast(
                        float, __builtin_amdgcn_raw_buffer_load_b32(rb, 4 * (n - nw + 8 * (r >> 2) + (r & 3)), 0, 0));
                __builtin_amdgcn_s_waitcnt(MX4_WAIT(0));  // (here, not where the sides meet)
            }
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t at = (uint32_t)(wm + 32 * i + (lane & 31)) * (uint32_t)a.N;
                float v[16];
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    v[r] = acc[i][j][r] + bias[r >> 2][r & 3];
                    if (GELU) v[r] = gelu_tanh(v[r]);
                }
                auto to = [&](int c) { return c < a.N ? (at + c) * E : ~0u; };
                if constexpr (!WIDE) {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const uint32_t d = to(n + 8 * (r >> 2) + (r & 3));
                        if constexpr (E == 4)
                            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v[r]), ry, d, 0, 0);
                        else
                            __builtin_amdgcn_raw_buffer_store_b16(Op<Out>::bits(v[r]), ry, d, 0, 0);
                    }
                } else if constexpr (E == 4) {
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        __builtin_amdgcn_raw_buffer_store_b128(
                            __builtin_bit_cast(u32x4, (f32x4){v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]}), ry,
                            to(n + 8 * g), 0, 0);
                } else {
#pragma unroll
                    for (int g = 0; g < 4; g += 2) {
                        const auto p = __builtin_amdgcn_permlane32_swap(
                            Op<Out>::cvt2(v[4 * g], v[4 * g + 1]), Op<Out>::cvt2(v[4 * g + 4], v[4 * g + 5]), false, false);
                        const auto q = __builtin_amdgcn_permlane32_swap(Op<Out>::cvt2(v[4 * g + 2], v[4 * g + 3]),
                                                                        Op<Out>::cvt2(v[4 * g + 6], v[4 * g + 7]), false,
                                                                        false);
                        __builtin_amdgcn_raw_buffer_store_b128(
                            u32x4{(uint32_t)p[0], (uint32_t)q[0], (uint32_t)p[1], (uint32_t)q[1]}, ry,
                            to(n + 4 * h + 8 * g), 0, 0);
                    }
                }
            }
        }
    }

    // Resources that begin at the tile's first row (rows behind the last read as zeros), and
    // the DMA of its first two K-tiles (there false: of nothing, zeros).
    __device__ __forceinline__ void begin(int w, int m0, int n0, bool there) {
        const int G = a.K / 128, lane = threadIdx.x & 63;
        const uint32_t row = (uint32_t)a.K / 2;
        ra_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.a + (size_t)m0 * row), 0,
                                                there ? (int)((uint32_t)min(TM, a.M - m0) * row) : 0, MX4_RSRC_W3);
        rb_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (size_t)n0 * row), 0,
                                                there ? (int)((uint32_t)min(TM, a.N - n0) * row) : 0, MX4_RSRC_W3);
        const int rows = w < 2 ? a.M : a.N, first = w < 2 ? m0 : n0;
        rs_ = __builtin_amdgcn_make_buffer_rsrc((void*)((w < 2 ? a.as : a.ws) + 4 * (size_t)first), 0,
                                                there ? (int)(4u * ((uint32_t)G * (uint32_t)rows - (uint32_t)first)) : 0,
                                                MX4_RSRC_W3);
        gstep = 4u * (uint32_t)rows;
        gs = 4 * lane + (w & 1) * gstep;
        dma<0>(mx4_sofs(0));
        dma<1>(mx4_sofs(1));
    }

    __device__ __forceinline__ void run() {
        const int tid = threadIdx.x, lane = tid & 63;
        const int w = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;  // within the group
        kg = __builtin_amdgcn_readfirstlane(tid >> 8);
        const int wm = 32 * NB * (w >> 1), wn = 32 * NB * (w & 1);
        const int nk = 2 * ((a.K / 128 + 4 * KG - 1) / (4 * KG));
        lw = 1024 * ND * w + 128 * TM * kg;
        lsw = 4 * TM * w + 16 * TM * kg;
        {
            const int h = lane >> 5, r = lane & 31;
            off = (wm + r) * 128 + 16 * (h ^ ((r >> 1) & 7)) + 128 * TM * kg;
            ofw = (wn - wm) * 128;
            soff = 4 * (wm + r) + 16 * TM * kg;
            sofw = 8 * TM + 4 * (wn - wm);
            shift = 8 * h;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int tr = 8 * (ND * w + i) + (lane >> 3);
            ga[i] = (uint32_t)tr * ((uint32_t)a.K / 2) + 16u * ((lane & 7) ^ ((tr >> 1) & 7));
        }
        const int ntiles = a.tiles_m * a.tiles_n;
        auto tile_at = [&](int i) {  // (in scalar registers, whatever the compiler makes of the loop)
            const TileIdx t = tile_of(i, a.tiles_m, a.tiles_n);
            return TileIdx{__builtin_amdgcn_readfirstlane(t.tm), __builtin_amdgcn_readfirstlane(t.tn)};
        };
        int item = blockIdx.x;
        TileIdx ti = tile_at(item);
        begin(w, ti.tm * TM, ti.tn * TM, true);
        meet();
        while (true) {
            // the tile's first two K-tiles have landed for all waves
            region<4, 0, 0, 0>(0, 0, 0);
            region<0, 0, 1, 0, true>(0, 0, 0);
            region<1, 0, 2, 0>(0, 0, 0);
            region<2, 0, 3, 0>(0, 0, 0);
            meet<false>();
            for (int k = 0; k < nk - 2; k += 2) {
                tile<0, true>(k);
                tile<1, true>(k + 1);
            }
            const int m0 = ti.tm * TM, n0 = ti.tn * TM + wn;
            const __amdgpu_buffer_rsrc_t ry = __builtin_amdgcn_make_buffer_rsrc(
                (void*)((Out*)a.y + (size_t)m0 * a.N), 0,
                (int)((uint32_t)min(TM, a.M - m0) * (uint32_t)a.N * (uint32_t)sizeof(Out)), MX4_RSRC_W3);
            if constexpr (KG > 1) {  // (a tile a workgroup)
                tile<0, false>(nk - 2);
                region<3, 0, 4, 0>(0, 0, 0);
                if (!sum_groups(w)) return;
                store(ry, wm, n0);
                return;
            }
            item += gridDim.x;
            const bool more = item < ntiles;
            ti = tile_at(more ? item : (int)blockIdx.x);
            tile<0, false>(nk - 2);
            // Every wave has what is left in registers: the next tile's operands come in while
            // it is multiplied and y is formed, and y's stores leave beside the next tile.
            // (Behind the last tile no operand is read.)
            begin(w, ti.tm * TM, ti.tn * TM, more);
            __builtin_amdgcn_sched_barrier(0);
            region<3, 0, 4, 0>(0, 0, 0);
            hold();
            // the stores come behind the DMA, in order: it has landed when only they are left
            // (the counter's 63 would be no wait)
            constexpr int stores = NB * NB * (!WIDE ? 16 : sizeof(Out) == 4 ? 4 : 2);
            store(ry, wm, n0);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(MX4_WAIT(stores < 62 ? stores : 62));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            if (!more) break;
        }
    }
};

#define MX4_GEMM_KERNEL(NAME, OUT_, NB_, GELU_, WIDE_, KG_, PER_)                                   \
    extern "C" __global__ void __launch_bounds__(256 * KG_, PER_) NAME(const LtxMx4LinearArgs a) { \
        Mx4Gemm<OUT_, NB_, GELU_, WIDE_, KG_> k(a);                                                \
        k.run();                                                                                   \
    }
