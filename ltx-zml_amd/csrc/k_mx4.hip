// Microscaled 4-bit operands (the form of ltx_args.h): rows into it and back, and the
// linear of few rows.
#include <type_traits>

#include "gemm_mx4.h"

// ---- rows ---------------------------------------------------------------------------
// A wave takes 32 rows of 128 k, 16 lanes of eight values a row, four rows at a time. So
// that no access is smaller than it must be, the lanes of a quad exchange the codes of
// four times four rows: each stores 16 bytes, a whole group's, and the scale codes of 16
// rows are 64 bytes next to each other. Bound by memory: 28,672 x 4,096 f16 rows (235 MB
// in, 62 out) in 68 us, 4.4 TB/s, and back in 52; eight rows are a launch, 3 us each way.
template <typename T>
struct Mx4Rows;  // eight values of a row
template <>
struct Mx4Rows<float> {
    f32x4 x[2];
    __device__ __forceinline__ void load(const void* p, size_t at) {
        x[0] = *(const f32x4*)((const float*)p + at);
        x[1] = *(const f32x4*)((const float*)p + at + 4);
    }
    __device__ __forceinline__ void zero() { x[0] = x[1] = f32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ uint32_t encode(uint32_t& code) const {
        const float v[8] = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
        return fp4_encode<float>(v, code);
    }
    static __device__ __forceinline__ void store(void* p, size_t at, const float (&v)[8]) {
        *(f32x4*)((float*)p + at) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)((float*)p + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
};
template <typename T>
struct Mx4Rows {
    u32x4 x;
    __device__ __forceinline__ void load(const void* p, size_t at) { x = *(const u32x4*)((const uint16_t*)p + at); }
    __device__ __forceinline__ void zero() { x = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ uint32_t encode(uint32_t& code) const { return fp4_encode<T>(x, code); }
    static __device__ __forceinline__ void store(void* p, size_t at, const float (&v)[8]) {
        *(u32x4*)((uint16_t*)p + at) = u32x4{Op<T>::cvt2(v[0], v[1]), Op<T>::cvt2(v[2], v[3]), Op<T>::cvt2(v[4], v[5]),
                                             Op<T>::cvt2(v[6], v[7])};
    }
};

template <typename T>
__device__ __forceinline__ void mx4_quantise(const LtxMx4RowsArgs& a) {
    const int G = a.K / 128, across = (G + 3) / 4;
    const int lane = threadIdx.x & 63, o = lane & 15, sub = lane >> 4;
    const int by = blockIdx.x / across, kg = 4 * (blockIdx.x - by * across) + (threadIdx.x >> 6);
    const int row0 = 32 * by;
    if (kg >= G) return;
    Mx4Rows<T> x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int row = row0 + 4 * e + sub;
        x[e].zero();
        if (row < a.rows) x[e].load(a.x, (size_t)row * a.ldx + 128 * kg + 8 * o);
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
        u32x4 q, c;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint32_t code;
            q[e] = x[4 * b + e].encode(code);
            c[e] = code;
        }
        quad_transpose(q);
        const uint32_t code = quad_pick(c);
        const int row = row0 + 16 * b + 4 * (o & 3) + sub;
        if (row < a.rows) {
            *(u32x4*)(a.q + (size_t)row * (a.K / 2) + 64 * kg + 16 * (o >> 2)) = q;
            a.s[((size_t)kg * a.rows + row) * 4 + (o >> 2)] = (uint8_t)code;
        }
    }
}

// Code times 2^(scale code - 127), rounded to the type.
template <typename T>
__device__ __forceinline__ void mx4_values(const LtxMx4RowsArgs& a) {
    const int G = a.K / 128, across = (G + 3) / 4;
    const int lane = threadIdx.x & 63, o = lane & 15, sub = lane >> 4;
    const int by = blockIdx.x / across, kg = 4 * (blockIdx.x - by * across) + (threadIdx.x >> 6);
    if (kg >= G) return;
    uint32_t q[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int row = 32 * by + 4 * e + sub;
        q[e] = s[e] = 0;
        if (row < a.rows) {
            q[e] = *(const uint32_t*)(a.q + (size_t)row * (a.K / 2) + 64 * kg + 4 * o);
            s[e] = a.s[((size_t)kg * a.rows + row) * 4 + (o >> 2)];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int row = 32 * by + 4 * e + sub;
        if (row >= a.rows) continue;
        const float nan = s[e] == 255u ? __builtin_nanf("") : 0.f;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // a code is 2^(exponent - 1) (1 + mantissa / 2), or mantissa / 2
            const uint32_t c = q[e] >> (4 * i), m = c & 1u, x = (c >> 1) & 3u;
            const float y = x ? (float)((2 + m) << x) * 0.25f : 0.5f * (float)m;
            v[i] = ldexpf(c & 8u ? -y : y, (int)s[e] - 127) + nan;
        }
        Mx4Rows<T>::store(a.x, (size_t)row * a.ldx + 128 * kg + 8 * o, v);
    }
}

#define MX4_ROWS(NAME, FN, T) \
    extern "C" __global__ void __launch_bounds__(256) NAME(const LtxMx4RowsArgs a) { FN<T>(a); }
MX4_ROWS(ltx_mx4_quantise_f16, mx4_quantise, _Float16)
MX4_ROWS(ltx_mx4_quantise_bf16, mx4_quantise, __bf16)
MX4_ROWS(ltx_mx4_quantise_f32, mx4_quantise, float)
MX4_ROWS(ltx_mx4_values_f16, mx4_values, _Float16)
MX4_ROWS(ltx_mx4_values_bf16, mx4_values, __bf16)
MX4_ROWS(ltx_mx4_values_f32, mx4_values, float)

// ---- the linear of few rows -----------------------------------------------------------
// A workgroup takes 16 MT rows of a and 16 NT of w (columns of y); its eight waves take
// pairs of steps of 128 k in turn (a line of w's codes), straight from memory into the
// registers of v_mfma_scale_f32_16x16x128_f8f6f4, whose operand is a lane's 16 bytes and
// scale code: w is read once and never leaves its form. The waves' sums are added in their
// order. ROWS: a holds 16-bit values, and each lane makes the group of 32 that it
// multiplies from 64 bytes of its row: nothing crosses lanes, and one row of a model's
// linear is one launch. Bound by that launch (3.8 us of 5.1 for one row of 4,096 x 4,096,
// whose 8.9 MB are 1.8) and by w's bytes as N grows.
#define MX4_WAVES 8

template <typename T>
__device__ __forceinline__ u32x4 mx4_group(const u32x4 (&x)[4], uint32_t& code) {
    u16x2 top = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t y = x[j][e] & 0x7fff7fffu;
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, y));
        }
    const float t = Op<T>::to_f32(top[0] > top[1] ? top[0] : top[1]);
    code = fp4_code<T>(__builtin_bit_cast(uint32_t, t));
    const float s = __builtin_bit_cast(float, code << 23);
    u32x4 q;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t y = 0;
        auto put = [&](auto E) {
            constexpr int e = decltype(E)::value;
            const uint32_t w = x[j][e];
            if constexpr (__is_same(T, _Float16))
                y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(y, __builtin_bit_cast(f16x2, w), s, e);
            else
                y = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(y, __builtin_bit_cast(bf16x2, w), s, e);
        };
        put(std::integral_constant<int, 0>{});
        put(std::integral_constant<int, 1>{});
        put(std::integral_constant<int, 2>{});
        put(std::integral_constant<int, 3>{});
        q[j] = y;
    }
    return q;
}

template <typename T, bool ROWS, int MT, int NT>
__device__ __forceinline__ void mx4_few(const LtxMx4LinearArgs& a) {
    constexpr int D = MT == 1 ? 4 : ROWS && MT * NT == 16 ? 1 : 2, NA = ROWS ? 4 : 1;  // steps in flight
    __shared__ __attribute__((aligned(16))) float sums[MX4_WAVES][MT * NT][64][4];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = 16 * MT * blockIdx.y, n0 = 16 * NT * blockIdx.x;
    const int rows = min(16 * MT, a.M - m0), cols = min(16 * NT, a.N - n0), G = a.K / 128;
    const uint32_t lw = (uint32_t)a.K / 2, la = ROWS ? 4 * lw : lw;  // bytes of a row
    // resources that begin at the workgroup's first rows and end behind its last (the scale
    // words': behind those of the last group): what lies past them reads as zeros. Rows past
    // the last have codes of 0, whatever scale words they meet.
    auto rsrc = [](const void* p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, MX4_RSRC_W3);
    };
    const __amdgpu_buffer_rsrc_t ra = rsrc(a.a + (size_t)m0 * la, rows * la), rw = rsrc(a.w + (size_t)n0 * lw, cols * lw);
    const __amdgpu_buffer_rsrc_t rsa =
        rsrc(ROWS ? a.w : a.as + 4 * (size_t)m0, ROWS ? 0 : 4u * ((uint32_t)G * a.M - m0));
    const __amdgpu_buffer_rsrc_t rsw = rsrc(a.ws + 4 * (size_t)n0, 4u * ((uint32_t)G * a.N - n0));
    // Steps in flight: w's of D, a's of as many where they are codes or one tile, else of one,
    // whose tiles make way for the next step's one by one.
    constexpr int DA = ROWS && MT > 1 ? 1 : D;
    u32x4 xa[DA][MT][NA], xw[D][NT];
    uint32_t sa[DA][MT], sw[D][NT];
    auto step = [&](int i) { return 2 * (w + MX4_WAVES * (i >> 1)) + (i & 1); };
    auto load_a = [&](int d, int m, int g) {
        if (g >= G) return;
#pragma unroll
        for (int j = 0; j < NA; j++)
            xa[d][m][j] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, (16 * m + r) * la + (ROWS ? 64 : 16) * h + 16 * j,
                                                             (ROWS ? 256 : 64) * g, 0));
        if (!ROWS) sa[d][m] = __builtin_amdgcn_raw_buffer_load_b8(rsa, 4 * (16 * m + r) + h + 4 * g * a.M, 0, 0);
    };
    auto load_w = [&](int d, int g) {
        if (g >= G) return;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            xw[d][t] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, (16 * t + r) * lw + 16 * h, 64 * g, 0));
            sw[d][t] = __builtin_amdgcn_raw_buffer_load_b8(rsw, 4 * (16 * t + r) + h + 4 * g * a.N, 0, 0);
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D; i++) {
        load_w(i, step(i));
        if (i < DA)
#pragma unroll
            for (int m = 0; m < MT; m++) load_a(i, m, step(i));
    }
#pragma nounroll
    for (int i = 0; step(i) < G; i += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            if (step(i + d) >= G) break;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                constexpr int last = DA - 1;
                const int e = d < DA ? d : last;
                u32x4 y = xa[e][m][0];
                if constexpr (ROWS) y = mx4_group<T>(xa[e][m], sa[e][m]);
                const uint32_t s = sa[e][m];
                __builtin_amdgcn_sched_barrier(0);
                load_a(e, m, step(i + d + DA));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = mx4_mfma16(y, xw[d][t], acc[m][t], s, sw[d][t]);
            }
            load_w(d, step(i + d + D));
        }
    }
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) *(f32x4*)sums[w][m * NT + t][lane] = acc[m][t];
    __syncthreads();
    for (int e = tid; e < MT * NT * 256; e += 64 * MX4_WAVES) {
        // column of the tile fastest: rows of y are written whole
        const int t = (e >> 4) % NT, row = (e >> 4) / NT, col = e & 15, n = n0 + 16 * t + col;
        if (row >= rows || n >= a.N) continue;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < MX4_WAVES; j++) y += sums[j][(row >> 4) * NT + t][16 * ((row & 15) >> 2) + col][row & 3];
        if (a.bias) y += a.bias[n];
        if (a.gelu) y = gelu_tanh(y);
        const size_t at = (size_t)(m0 + row) * a.N + n;
        if (a.out_f32)
            ((float*)a.y)[at] = y;
        else
            ((uint16_t*)a.y)[at] = Op<T>::bits(y);
    }
}

#define MX4_FEW(NAME, T, ROWS, MT, NT)                                                                     \
    extern "C" __global__ void __launch_bounds__(512) NAME##MT##_##NT(const LtxMx4LinearArgs a) {          \
        mx4_few<T, ROWS, MT, NT>(a);                                                                       \
    }
#define MX4_FEW_TILES(NAME, T, ROWS, MT) MX4_FEW(NAME, T, ROWS, MT, 1) MX4_FEW(NAME, T, ROWS, MT, 2) MX4_FEW(NAME, T, ROWS, MT, 4)
#define MX4_FEW_TYPE(TYPE, T)                             \
    MX4_FEW(ltx_linear_mx4_##TYPE##_, T, false, 1, 1)         \
    MX4_FEW(ltx_linear_mx4_##TYPE##_, T, false, 1, 2)         \
    MX4_FEW(ltx_linear_mx4_##TYPE##_, T, false, 2, 1)         \
    MX4_FEW_TILES(ltx_linear_mx4_##TYPE##_rows_, T, true, 1)  \
    MX4_FEW_TILES(ltx_linear_mx4_##TYPE##_rows_, T, true, 2)  \
    MX4_FEW_TILES(ltx_linear_mx4_##TYPE##_rows_, T, true, 3)  \
    MX4_FEW_TILES(ltx_linear_mx4_##TYPE##_rows_, T, true, 4)
MX4_FEW_TYPE(f16, _Float16)
MX4_FEW_TYPE(bf16, __bf16)
