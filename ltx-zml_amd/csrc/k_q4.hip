// y = a . (q s)^T (+ bias, GELU) with 4-bit weights, two a byte, and a scale per
// 128 along k: the linear of few rows.
#include <type_traits>

#include "ltx_device.h"

// Eight weights of a dword (two's complement nibbles, the lowest first) as 16-bit
// operands of value q / 16: v_cvt_off_f32_i4 (of the low four bits, exact) takes any
// byte of its operand, so that a shift serves the four odd nibbles; the rounding is
// exact too. 13 instructions. X: q / 1,024, six off the exponents of a pair (a zero's
// stays zero: the subtraction saturates).
template <typename T, bool X>
__device__ __forceinline__ u32x4 q4_operand(uint32_t w) {
    uint32_t o = w >> 4;
    asm("" : "+v"(o));  // one shift, not one an odd nibble
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++)
        r[e] = Op<T>::cvt2(__builtin_amdgcn_cvt_off_f32_i4((w >> (8 * e)) & 0xffu),
                           __builtin_amdgcn_cvt_off_f32_i4((o >> (8 * e)) & 0xffu));
    if (X) {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t x = r[e];
            r[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, x), (u16x2)(6 << 7)));
        }
    }
    return r;
}

#define Q4_WAVES 8

// Operands come through buffer resources that begin at the workgroup's first row:
// rows past the last read as zeros without an access. The group goes into the scalar
// offset, which takes no part in that check; for a group that is not there the
// resource is empty instead. So the loads need no branch and no vector arithmetic.
typedef __amdgpu_buffer_rsrc_t q4_rsrc;
struct Q4Buffer {
    const void* base;
    int bytes;
    __device__ __forceinline__ q4_rsrc rsrc(bool there) const {
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, there ? bytes : 0, 0x00020000);
    }
};
__device__ __forceinline__ u32x4 q4_load16(q4_rsrc b, uint32_t lane, uint32_t all) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, lane, all, 0));
}
template <bool S16>
__device__ __forceinline__ uint32_t q4_load_scale(q4_rsrc b, uint32_t lane, uint32_t all) {
    return S16 ? (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(b, 2 * lane, 2 * all, 0)
               : (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b, 4 * lane, 4 * all, 0);
}
template <bool S16>
__device__ __forceinline__ float q4_scale(uint32_t bits) {
    return S16 ? f16_bits_to_f32((uint16_t)bits) : __builtin_bit_cast(float, bits);
}

// The waves' sums into one, in the waves' order, and y. my: the wave's slot of SLOT
// bytes in lds. IN: rows of D that make a row of y.
template <typename T, int MT, int NT, int SLOT, int IN>
__device__ __forceinline__ void q4_finish(const LtxLinearQ4Args& a, uint8_t* lds, int w, int lane,
                                          const f32x4 (&acc)[MT][NT], int m0, int n0, int rows) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) *(f32x4*)(lds + SLOT * w + 1024 * (m * NT + t) + 16 * lane) = acc[m][t];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * NT * 256; e += 64 * Q4_WAVES) {
        // element e: column of the tile fastest, so that rows of y are written whole
        const int t = (e >> 4) % NT, row = (e >> 4) / NT, col = e & 15, m = row >> 4;
        const int n = n0 + 16 * t + col;
        if (row >= rows || n >= a.N) continue;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < Q4_WAVES; j++)
#pragma unroll
            for (int i = 0; i < IN; i++) {
                const int d = IN * row + i;
                y += *(const float*)(lds + SLOT * j + 1024 * (m * NT + t) + 16 * (16 * ((d & 15) >> 2) + col) +
                                     4 * (d & 3));
            }
        y *= 16.0f;  // of the operands
        if (a.bias) y += a.bias[n];
        if (a.gelu) y = gelu_tanh(y);
        const size_t at = (size_t)(m0 + row) * a.N + n;
        if (a.out_f32)
            ((float*)a.y)[at] = y;
        else
            ((uint16_t*)a.y)[at] = Op<T>::bits(y);
    }
}

// The scales of four groups, group h's in lanes 16 h .. + 15, to all lanes each.
__device__ __forceinline__ void q4_spread(uint32_t x, uint32_t (&s)[4]) {
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);  // groups 0 1 0 1 and 2 3 2 3
    auto b = __builtin_amdgcn_permlane16_swap(a[0], a[0], false, false);
    s[0] = b[0], s[1] = b[1];
    b = __builtin_amdgcn_permlane16_swap(a[1], a[1], false, false);
    s[2] = b[0], s[3] = b[1];
}

// Four values as three bf16 planes, x = p0 + p1 + p2 exactly from 2^-110 on (the lowest
// plane ends at bf16's smallest subnormal; split3 of the f32 GEMM, four at a time).
__device__ __forceinline__ void q4_split(f32x4 x, u32x2 (&p)[3]) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float v = x[e];  // (a bit cast of a vector's element itself takes element 0)
        h[e] = __builtin_bit_cast(uint32_t, v) & 0xffff0000u;
        const float d = __builtin_isinf(v) ? 0.0f : v - __builtin_bit_cast(float, h[e]);
        m[e] = __builtin_bit_cast(uint32_t, d) & 0xffff0000u;
        l[e] = __builtin_bit_cast(uint32_t, d - __builtin_bit_cast(float, m[e]));
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
        p[0][e] = __builtin_amdgcn_perm(h[2 * e + 1], h[2 * e], 0x07060302u);
        p[1][e] = __builtin_amdgcn_perm(m[2 * e + 1], m[2 * e], 0x07060302u);
        p[2][e] = __builtin_amdgcn_perm(l[2 * e + 1], l[2 * e], 0x07060302u);
    }
}

// A workgroup takes 16 MT rows of a and 16 NT of q, each of its eight waves an
// eighth of the groups of 128. PLANES: the exact planes that make a value of a, three
// in mode F32. PACK: they are rows of one tile, 3 row + plane, summed with the waves'
// parts at the end, where up to five rows of a leave it place. D's column is the weight
// row, so a lane needs one scale of a group, which multiplies the group's f32 sum.
//
// Bound: the weights, read once, 4,096 x 4,096 in 2 us at the rate of a large copy
// (4.9 TB/s). MFMA operands want neighbouring lanes in different rows; loaded that
// way every lane is an access of its own, 64 an instruction where 16 would do, and
// the texture unit bounds the kernel (16 rows of 16,384 x 4,096: 12.6 million
// accesses, 30 us; with scalar offsets in place of a third of the vector
// instructions no faster). So both operands are loaded along their rows and change
// lanes in LDS of the wave's own (no barrier, and the order of a wave's LDS
// operations lets one buffer do): chunk c (16 bytes) of row r of a at c ^ r, of q at
// c ^ r / 2, free of conflicts. AW groups of q and AA of a are in flight.
// Measured back to back in a graph, where an empty launch takes 3.8 us: one row 5.7
// us (4,096 x 4,096), 10.4 (16,384 x 4,096), 10.4 (4,096 x 16,384); 32 rows of
// 16,384 x 4,096 14.3 us (bf16; 17.5 with NT = 2, 21.1 with MT = 1); mode F32, one row of
// 4,096 x 16,384 11.4 us, five 15.7 (without PACK 15.9 and 20.2: three times the LDS
// reads and products; what five rows take beyond one is every workgroup's reading and
// splitting of all of them).
template <typename T, int PLANES, bool PACK, bool S16, int MT, int NT, int AW, int AA, int EARLY>
__device__ __forceinline__ void linear_q4(const LtxLinearQ4Args& a) {
    typedef typename Op<T>::v8 v8;
    constexpr bool F32 = PLANES == 3;
    constexpr int PL = PACK ? 1 : PLANES;  // of them in tiles of their own
    constexpr int XT = MT * PL * 4096, TILE = XT + NT * 1024, PART = MT * NT * 1024;
    constexpr int SLOT = TILE > PART ? TILE : PART;
    __shared__ __attribute__((aligned(16))) uint8_t lds[Q4_WAVES * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int rows = min(16 * MT, a.M - m0), cols = min(16 * NT, a.N - n0);
    const int G = a.K / LTX_GROUP, each = (G + Q4_WAVES - 1) / Q4_WAVES;
    const int g0 = w * each, g1 = min(G, g0 + each);
    uint8_t* my = lds + w * SLOT;
    const Q4Buffer bq{a.q + (size_t)n0 * (a.K / 2), cols * (a.K / 2)};
    const Q4Buffer bs{(const char*)a.scales + (size_t)n0 * G * (S16 ? 2 : 4), cols * G * (S16 ? 2 : 4)};
    const Q4Buffer bx{(const char*)a.a + (size_t)m0 * a.K * (F32 ? 4 : 2), rows * a.K * (F32 ? 4 : 2)};
    // loads: q chunk l % 4 of row l / 4; a chunk l % 16 (8 values) of rows 4 i + l / 16
    const uint32_t oq = (lane >> 2) * (a.K / 2) + 16 * (lane & 3), os = r * G + h;
    const uint32_t ox = F32 ? (lane >> 5) * 4 * a.K + 16 * (lane & 31) : h * 2 * a.K + 16 * r;
    uint8_t* wq_st = my + XT + 64 * (lane >> 2) + 16 * ((lane & 3) ^ ((lane >> 3) & 3));
    const uint8_t* wq_ld = my + XT + 64 * r + 16 * (h ^ ((r >> 1) & 3));

    constexpr int NX = PACK ? 3 : F32 ? 8 * MT : 4 * MT, RX = F32 ? 2 : 4;  // loads of a group of a, rows of a load
    u32x4 wq[AW][NT], xa[AA][NX];
    uint32_t sc[NT];
    auto load_w = [&](int u, int g) {
        const q4_rsrc rq = bq.rsrc(g < g1);
#pragma unroll
        for (int t = 0; t < NT; t++) wq[u][t] = q4_load16(rq, oq + 16 * t * (a.K / 2), 64 * g);
    };
    auto load_s = [&](int g) {  // groups g .. g + 3, zero past the wave's last one
#pragma unroll
        for (int t = 0; t < NT; t++)
            sc[t] = q4_load_scale<S16>(bs.rsrc(g < g1), g + h < g1 ? os + 16 * t * G : 0x20000000u, g);
    };
    auto load_a = [&](int u, int g) {
        const q4_rsrc rx = bx.rsrc(g < g1);
#pragma unroll
        for (int i = 0; i < NX; i++) xa[u][i] = q4_load16(rx, ox + 8 * i * a.K, (F32 ? 512 : 256) * g);
    };
    struct Frags {
        u32x4 w[NT];
        v8 x[MT][PL][4];
    };
    auto exchange = [&](int u, Frags& f) {
#pragma unroll
        for (int t = 0; t < NT; t++) *(u32x4*)(wq_st + 1024 * t) = wq[u % AW][t];
#pragma unroll
        for (int i = 0; i < NX; i++) {
            if (RX * i >= rows) continue;
            if (F32) {
                const int row = 2 * i + (lane >> 5), c = lane & 31;
                u32x2 p[3];
                q4_split(__builtin_bit_cast(f32x4, xa[u % AA][i]), p);
                if (PACK && row >= LTX_Q4_PACKED) continue;
#pragma unroll
                for (int j = 0; j < 3; j++) {
                    const int at = PACK ? 3 * row + j : row;
                    *(u32x2*)(my + (PACK ? 0 : 4096 * MT * j) + 256 * at + 16 * ((c >> 1) ^ (at & 15)) +
                              8 * (c & 1)) = p[j];
                }
            } else {
                const int row = 4 * i + h;
                *(u32x4*)(my + 256 * row + 16 * (r ^ (row & 15))) = xa[u % AA][i];
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) f.w[t] = *(const u32x4*)(wq_ld + 1024 * t);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int p = 0; p < PL; p++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    f.x[m][p][j] = __builtin_bit_cast(
                        v8, *(const u32x4*)(my + 4096 * (MT * p + m) + 256 * r + 16 * ((4 * h + j) ^ r)));
    };
    // acc = the wave's groups; X: with weights times 2^-6 and scales times 2^6
    auto sums = [&](auto x, f32x4 (&acc)[MT][NT]) {
        constexpr bool X = decltype(x)::value;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < NT; t++) acc[m][t] = f32x4{0, 0, 0, 0};

        load_s(g0);
#pragma unroll
        for (int u = 0; u < AW; u++) {
            load_w(u, g0 + u);
            if (u < AA) load_a(u, g0 + u);
            __builtin_amdgcn_sched_barrier(0);
        }
        // EARLY 1: a group's exchange runs before the products of the one before it
        Frags f[1 + EARLY];
        if (EARLY) {
            exchange(0, f[0]);
            load_w(0, g0 + AW);
            load_a(0, g0 + AA);
        }
        for (int g = g0; g < g1; g += AW) {
            uint32_t sg[NT][4];
#pragma unroll
            for (int t = 0; t < NT; t++) q4_spread(sc[t], sg[t]);
            load_s(g + AW);
#pragma unroll
            for (int u = 0; u < AW; u++) {
                exchange(u + EARLY, f[(u + EARLY) & EARLY]);
                // the loads stay here: gathered behind all of the step's products they
                // would be waited for all at once
                load_w((u + EARLY) % AW, g + u + EARLY + AW);
                load_a((u + EARLY) % AA, g + u + EARLY + AA);
                f32x4 d[MT][NT];
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int t = 0; t < NT; t++) d[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const v8 wv = __builtin_bit_cast(v8, q4_operand<T, X>(f[u & EARLY].w[t][j]));
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int p = 0; p < PL; p++) d[m][t] = Op<T>::mfma16(f[u & EARLY].x[m][p][j], wv, d[m][t]);
                    }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float s = X ? 64.0f * q4_scale<S16>(sg[t][u]) : q4_scale<S16>(sg[t][u]);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[m][t][i] = __builtin_fmaf(d[m][t][i], s, acc[m][t][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    f32x4 acc[MT][NT];
    sums(std::false_type{}, acc);
    // A group's sum of a q / 16 may leave f32's range, from |a| = 2^122 on, where y does
    // not. A wave with a sum that is not finite forms its sums once more with the weights
    // times 2^-6, whose products are no larger than a, and the scales times 2^6 (exact below 2^122): the
    // range is that of a and y, and an infinity or NaN in a stays one. (f16 values are
    // too small for that.)
    if constexpr (__is_same(T, __bf16)) {
        float worst = 0.f;  // 0, or NaN
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)  // (rows of D past the last may hold anything)
                    if (16 * m + 4 * h + i < (PACK ? 3 * rows : rows)) worst = __builtin_fmaf(acc[m][t][i], 0.f, worst);
        if (__builtin_amdgcn_ballot_w64(worst != 0.f)) sums(std::true_type{}, acc);
    }
    q4_finish<T, MT, NT, SLOT, PACK ? 3 : 1>(a, lds, w, lane, acc, m0, n0, rows);
}

#define Q4_KERNEL(NAME, ...)                                                                        \
    extern "C" __global__ void __launch_bounds__(64 * Q4_WAVES) NAME(const LtxLinearQ4Args a) {    \
        linear_q4<__VA_ARGS__>(a);                                                                  \
    }
#define Q4_KERNELS(MT, NT, ...)                                                           \
    Q4_KERNEL(ltx_linear_q4_f16_s32_##MT##_##NT, _Float16, 1, false, false, MT, NT, __VA_ARGS__) \
    Q4_KERNEL(ltx_linear_q4_f16_s16_##MT##_##NT, _Float16, 1, false, true, MT, NT, __VA_ARGS__)  \
    Q4_KERNEL(ltx_linear_q4_bf16_s32_##MT##_##NT, __bf16, 1, false, false, MT, NT, __VA_ARGS__)  \
    Q4_KERNEL(ltx_linear_q4_bf16_s16_##MT##_##NT, __bf16, 1, false, true, MT, NT, __VA_ARGS__)
#define Q4_PLANES(MODE, PACK, NT, ...)                                                             \
    Q4_KERNEL(ltx_linear_q4_##MODE##_s32_1_##NT, __bf16, 3, PACK, false, 1, NT, __VA_ARGS__)       \
    Q4_KERNEL(ltx_linear_q4_##MODE##_s16_1_##NT, __bf16, 3, PACK, true, 1, NT, __VA_ARGS__)
Q4_KERNELS(1, 1, 4, 4, 1)
Q4_KERNELS(1, 2, 4, 4, 1)
Q4_KERNELS(1, 4, 4, 2, 0)
Q4_KERNELS(2, 1, 4, 2, 1)
Q4_KERNELS(2, 2, 4, 2, 0)
Q4_KERNELS(2, 4, 2, 1, 0)
Q4_PLANES(f32, false, 1, 4, 2, 1)
Q4_PLANES(f32, false, 2, 4, 2, 0)
Q4_PLANES(f32, false, 4, 4, 1, 0)
Q4_PLANES(f32p, true, 1, 4, 4, 1)
Q4_PLANES(f32p, true, 2, 4, 4, 1)
Q4_PLANES(f32p, true, 4, 4, 2, 0)
