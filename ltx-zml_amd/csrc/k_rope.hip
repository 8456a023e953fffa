// Norm and rotary positions of q and k on several axes.
#include <type_traits>

#include "ltx_device.h"

// Eight values of a row.
template <typename T>
struct RopeRow {
    u32x4 x;
    __device__ __forceinline__ void load(const void* p, size_t at) { x = *(const u32x4*)((const uint16_t*)p + at); }
    __device__ __forceinline__ float get(int e) const { return Op<T>::to_f32((uint16_t)(x[e >> 1] >> (16 * (e & 1)))); }
    static __device__ __forceinline__ void store(void* p, size_t at, const float (&v)[8]) {
        *(u32x4*)((uint16_t*)p + at) = u32x4{Op<T>::cvt2(v[0], v[1]), Op<T>::cvt2(v[2], v[3]), Op<T>::cvt2(v[4], v[5]),
                                             Op<T>::cvt2(v[6], v[7])};
    }
};
template <>
struct RopeRow<float> {
    f32x4 x[2];
    __device__ __forceinline__ void load(const void* p, size_t at) {
        x[0] = *(const f32x4*)((const float*)p + at);
        x[1] = *(const f32x4*)((const float*)p + at + 4);
    }
    __device__ __forceinline__ float get(int e) const { return x[e >> 2][e & 3]; }
    static __device__ __forceinline__ void store(void* p, size_t at, const float (&v)[8]) {
        *(f32x4*)((float*)p + at) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)((float*)p + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
};

// What eight pairs of a plan's head turn by: quarter turns a unit of position, at position
// 0, and the axes (a byte each).
struct RopePairs {
    double freq[8], phase[8];
    uint32_t axis[2];
    __device__ __forceinline__ void load(const LtxRopeArgs& a, int unit) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            freq[j] = a.freq[8 * unit + j];
            phase[j] = a.phase[8 * unit + j];
        }
        const u32x2 x = *(const u32x2*)(a.axis + 8 * unit);
        axis[0] = x[0];
        axis[1] = x[1];
    }
};

// cos and sin of t quarter turns. Angles go far (thousands of turns, where f32 holds no
// fraction of one), so whole quarters are taken off in f64: adding 1.5 2^52 rounds t to
// them, and leaves their last bits in the sum's (|t| below 2^51). What is left, within half a
// quarter, takes the series of sin and cos: their next terms are 1.8e-9 and 1.2e-10 there.
__device__ __forceinline__ void rope_turn(double t, float& c, float& s) {
    const double up = t + 6755399441055744.0;
    const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, up);
    const float x = (float)(t - (up - 6755399441055744.0)) * 1.57079632679489662f, z = x * x;
    float p = __builtin_fmaf(z, 2.755731922e-6f, -1.984126984e-4f);
    p = __builtin_fmaf(z, p, 8.333333333e-3f);
    p = __builtin_fmaf(z, p, -1.666666667e-1f);
    const float sx = __builtin_fmaf(x * z, p, x);
    float r = __builtin_fmaf(z, -2.755731922e-7f, 2.480158730e-5f);
    r = __builtin_fmaf(z, r, -1.388888889e-3f);
    r = __builtin_fmaf(z, r, 4.166666667e-2f);
    r = __builtin_fmaf(z, r, -0.5f);
    const float cx = __builtin_fmaf(z, r, 1.0f);
    // a quarter takes (c, s) to (-s, c)
    const float c0 = k & 1 ? sx : cx, s0 = k & 1 ? cx : sx;
    c = (k + 1) & 2 ? -c0 : c0;
    s = k & 2 ? -s0 : s0;
}

__device__ __forceinline__ void rope_turns(const RopePairs& p, const double* pos, float (&c)[8], float (&s)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        rope_turn(__builtin_fma(p.freq[j], pos[(p.axis[j >> 2] >> (8 * (j & 3))) & 255u], p.phase[j]), c[j], s[j]);
}

// The sums of squares of two rows over the workgroup (256 threads).
__device__ __forceinline__ void rope_sums(float& x, float& y, float (*red)[2]) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        x += __shfl_xor(x, o, 64);
        y += __shfl_xor(y, o, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6][0] = x;
        red[threadIdx.x >> 6][1] = y;
    }
    __syncthreads();
    x = red[0][0] + red[1][0] + red[2][0] + red[3][0];
    y = red[0][1] + red[1][1] + red[2][1] + red[3][1];
}

// A normed row is multiplied by 1 / sqrt(mean square + eps). Sums of squares are f32's; where that
// leaves it (f16's never do), the row's mean square is formed again in f64, and the row multiplied
// by a power of two near the root's inverse (`first`), then by the rest of it. `ms`: the same for
// the whole workgroup. What this costs where no row needs it: nothing up to 32 heads (28,672 rows of
// 32 + 32 bf16 heads 207 us with and without), beyond between 5 % (40 + 8 bf16 heads 468 -> 491)
// and -3 % (48 + 48 f32 heads, 14,336 rows, 625 -> 605).
template <typename T>
__device__ __forceinline__ bool rope_far(float ms) {
    return !__is_same(T, _Float16) && !(ms >= 0x1p-90f && ms <= __FLT_MAX__);
}
__device__ __forceinline__ float rope_far_factor(double sum, int n, float eps, float& first) {
    const double root = sqrt(sum / (double)n + (double)eps);
    const int e = -__builtin_amdgcn_frexp_exp(root), near = min(max(e, -126), 126);
    first = ldexpf(1.f, near);
    return ldexpf((float)(1.0 / __builtin_amdgcn_frexp_mant(root)), e - near);
}
// The sum over the workgroup of each thread's x.
__device__ __forceinline__ double rope_far_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// The sum over a wave's lanes, for all of them.
__device__ __forceinline__ float rope_wave_sum(float x) {
    auto add = [&](auto C, auto M) {
        const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(C)::value, decltype(M)::value, 0xf,
                                                  false);
        x += __builtin_bit_cast(float, y);
    };
    typedef std::integral_constant<int, 0xf> All;
    add(std::integral_constant<int, 0x111>{}, All{});
    add(std::integral_constant<int, 0x112>{}, All{});
    add(std::integral_constant<int, 0x114>{}, All{});
    add(std::integral_constant<int, 0x118>{}, All{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// Up to 32 heads, those of the set with fewer a divisor of the other's: thread t takes head
// h = t / 8 of the larger set, pairs 8 (t % 8) .. + 7, and of the other set head h / r where
// h is a multiple of r, their ratio: the plan's head of both, so one sine and cosine a pair
// serve both, and what the pairs turn by stays in registers (the weights in LDS) while the
// workgroup goes through its a.per rows. The next row's values are on their way while it
// works on one.
// Bound by memory: q and k of 28,672 rows, 32 + 32 f16 heads, normed, 940 MB in and out in
// 201 us, 4.7 TB/s, the rate of a copy (14,336 f32 rows the same). (With a workgroup a row, which loads the plan's
// 35 KB and the weights each time, 642.) 32 rows are a launch, 4.1 us.
template <typename T, bool NORM>
__device__ __forceinline__ void qk_rope_rows(const LtxRopeArgs& a) {
    __shared__ double spos[4][2][8];
    __shared__ float red[2][4][2];
    __shared__ double far[2][4];
    __shared__ f32x4 wt[NORM ? 2 : 1][4][256];  // a thread's own weights: in registers they cost a third of the waves
    const int h0 = threadIdx.x >> 3, o = threadIdx.x & 7, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int big = a.heads[1] > a.heads[0], ratio = a.heads[!big] ? a.heads[big] / a.heads[!big] : 1;
    const bool mine[2] = {h0 < a.heads[big], a.heads[!big] && h0 < a.heads[big] && h0 % ratio == 0};
    const int at[2] = {LTX_HD * h0 + 8 * o, LTX_HD * (h0 / ratio) + 8 * o};
    const int row0 = blockIdx.x * a.per, end = min(a.rows, row0 + a.per);
    RopePairs p;
    if (mine[0]) p.load(a, 8 * (h0 / a.group[big]) + o);
    if (NORM)
#pragma unroll
        for (int m = 0; m < 2; m++)
            if (const float* n = a.norm[m ^ big]; mine[m] && n)
#pragma unroll
                for (int j = 0; j < 4; j++) wt[m][j][threadIdx.x] = *(const f32x4*)(n + at[m] + 4 * (j & 1) + 64 * (j >> 1));
    RopeRow<T> x[2][2];
    double pos = 0;
    auto load = [&](int row) {
#pragma unroll
        for (int m = 0; m < 2; m++)
            if (mine[m]) {
                const size_t i = (size_t)row * a.ldx[m ^ big] + at[m];
                x[m][0].load(a.x[m ^ big], i);
                x[m][1].load(a.x[m ^ big], i + 64);
            }
        if (lane < a.axes) pos = a.pos[(size_t)row * a.axes + lane];
    };
    load(row0);
    for (int row = row0; row < end; row++) {
        float v[2][2][8], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 2; m++)
            if (mine[m])
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[m][0][j] = x[m][0].get(j);
                    v[m][1][j] = x[m][1].get(j);
                    if (NORM) {
                        sum[m] = __builtin_fmaf(v[m][0][j], v[m][0][j], sum[m]);
                        sum[m] = __builtin_fmaf(v[m][1][j], v[m][1][j], sum[m]);
                    }
                }
        // (a wave's own copy: its LDS operations come in order)
        if (lane < 8) spos[w][row & 1][lane] = pos;
        if (row + 1 < end) load(row + 1);
        if (NORM) {
            sum[0] = rope_wave_sum(sum[0]);
            sum[1] = rope_wave_sum(sum[1]);
            if (lane == 0) {
                red[row & 1][w][0] = sum[0];
                red[row & 1][w][1] = sum[1];
            }
        }
        float c[8], s[8];
        if (mine[0]) rope_turns(p, spos[w][row & 1], c, s);
        if (NORM) {
            __syncthreads();
#pragma unroll
            for (int m = 0; m < 2; m++) {
                if (!a.norm[m ^ big]) continue;
                const float all = red[row & 1][0][m] + red[row & 1][1][m] + red[row & 1][2][m] + red[row & 1][3][m];
                const float ms = all / (float)(LTX_HD * a.heads[m ^ big]) + a.eps;
                float inv = 1.0f / sqrtf(ms);
                if (rope_far<T>(ms)) {
                    double sum = 0;
                    if (mine[m])
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const double x = v[m][j >> 3][j & 7];
                            sum = __builtin_fma(x, x, sum);
                        }
                    float first;
                    // (the next row's sums come behind its barrier above)
                    inv = rope_far_factor(rope_far_sum(sum, far[m]), LTX_HD * a.heads[m ^ big], a.eps, first);
                    if (mine[m])
#pragma unroll
                        for (int j = 0; j < 16; j++) v[m][j >> 3][j & 7] *= first;
                }
                if (!mine[m]) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f32x4 n = wt[m][j][threadIdx.x];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[m][j >> 1][4 * (j & 1) + e] *= inv * n[e];
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2; m++) {
            if (!mine[m]) continue;
            float y[2][8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[0][j] = v[m][0][j] * c[j] - v[m][1][j] * s[j];
                y[1][j] = v[m][1][j] * c[j] + v[m][0][j] * s[j];
            }
            const size_t d = (size_t)row * a.ldy[m ^ big] + at[m];
            RopeRow<T>::store(a.y[m ^ big], d, y[0]);
            RopeRow<T>::store(a.y[m ^ big], d + 64, y[1]);
        }
    }
}

// Any heads: thread t takes head t / 8 and every 32nd after it. A row that is normed is read
// twice, and the plan again for every row. 28,672 f16 rows: 64 + 8 heads 285 us (3.7 TB/s), normed
// 705; normed 40 + 8 469, 48 + 48 951: 1.5 TB/s, where the kernel above runs at 4.7. 32 rows of 64 + 8
// 11.4.
template <typename T>
__device__ __forceinline__ void qk_rope(const LtxRopeArgs& a) {
    __shared__ float red[2][4][2];
    __shared__ double far[2][4];
    const int h0 = threadIdx.x >> 3, o = threadIdx.x & 7, at = 8 * o;
    const int row0 = blockIdx.x * a.per, end = min(a.rows, row0 + a.per);
    for (int row = row0; row < end; row++) {
        const double* pos = a.pos + (size_t)row * a.axes;
        float inv[2] = {1.f, 1.f}, first[2] = {1.f, 1.f};
        if (a.norm[0] || a.norm[1]) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; m++)
                if (a.norm[m])
                    for (int h = h0; h < a.heads[m]; h += 32) {
                        RopeRow<T> lo, hi;
                        const size_t i = (size_t)row * a.ldx[m] + LTX_HD * h + at;
                        lo.load(a.x[m], i);
                        hi.load(a.x[m], i + 64);
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            sum[m] = __builtin_fmaf(lo.get(j), lo.get(j), sum[m]);
                            sum[m] = __builtin_fmaf(hi.get(j), hi.get(j), sum[m]);
                        }
                    }
            rope_sums(sum[0], sum[1], red[row & 1]);
#pragma unroll
            for (int m = 0; m < 2; m++) {
                const int n = LTX_HD * max(a.heads[m], 1);
                const float ms = sum[m] / (float)n + a.eps;
                inv[m] = 1.0f / sqrtf(ms);
                if (!a.norm[m] || !rope_far<T>(ms)) continue;
                double all = 0;
                for (int h = h0; h < a.heads[m]; h += 32) {
                    RopeRow<T> x[2];
                    const size_t i = (size_t)row * a.ldx[m] + LTX_HD * h + at;
                    x[0].load(a.x[m], i);
                    x[1].load(a.x[m], i + 64);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const double y = x[j >> 3].get(j & 7);
                        all = __builtin_fma(y, y, all);
                    }
                }
                inv[m] = rope_far_factor(rope_far_sum(all, far[m]), n, a.eps, first[m]);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; m++)
            for (int h = h0; h < a.heads[m]; h += 32) {
                RopePairs p;
                p.load(a, 8 * (h / a.group[m]) + o);
                float c[8], s[8], u[8], v[8];
                rope_turns(p, pos, c, s);
                RopeRow<T> lo, hi;
                const size_t i = (size_t)row * a.ldx[m] + LTX_HD * h + at;
                lo.load(a.x[m], i);
                hi.load(a.x[m], i + 64);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float x = lo.get(j), y = hi.get(j);
                    if (a.norm[m]) {
                        if (!__is_same(T, _Float16)) {
                            x *= first[m];
                            y *= first[m];
                        }
                        x *= inv[m] * a.norm[m][LTX_HD * h + at + j];
                        y *= inv[m] * a.norm[m][LTX_HD * h + at + 64 + j];
                    }
                    u[j] = x * c[j] - y * s[j];
                    v[j] = y * c[j] + x * s[j];
                }
                const size_t d = (size_t)row * a.ldy[m] + LTX_HD * h + at;
                RopeRow<T>::store(a.y[m], d, u);
                RopeRow<T>::store(a.y[m], d + 64, v);
            }
    }
}

#define QK_ROPE(NAME, ...) \
    extern "C" __global__ void __launch_bounds__(256, 3) NAME(const LtxRopeArgs a) { __VA_ARGS__(a); }
QK_ROPE(ltx_qk_rope_f16, qk_rope_rows<_Float16, false>)
QK_ROPE(ltx_qk_rope_bf16, qk_rope_rows<__bf16, false>)
QK_ROPE(ltx_qk_rope_f32, qk_rope_rows<float, false>)
QK_ROPE(ltx_qk_rope_f16_norm, qk_rope_rows<_Float16, true>)
QK_ROPE(ltx_qk_rope_bf16_norm, qk_rope_rows<__bf16, true>)
QK_ROPE(ltx_qk_rope_f32_norm, qk_rope_rows<float, true>)
QK_ROPE(ltx_qk_rope_f16_any, qk_rope<_Float16>)
QK_ROPE(ltx_qk_rope_bf16_any, qk_rope<__bf16>)
QK_ROPE(ltx_qk_rope_f32_any, qk_rope<float>)
