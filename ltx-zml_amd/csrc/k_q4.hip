// y = a . (q s)^T (+ bias, GELU) with 4-bit weights, two a byte, and a scale per
// 128 along k: the linear of few rows.
#include "ltx_device.h"

// Eight weights of a dword (two's complement nibbles, the lowest first) as 16-bit
// operands of value q / 16: v_cvt_off_f32_i4 is exact, and so is the rounding.
template <typename T>
__device__ __forceinline__ u32x4 q4_operand(uint32_t w) {
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++)
        r[e] = Op<T>::cvt2(__builtin_amdgcn_cvt_off_f32_i4(w >> (8 * e)),
                           __builtin_amdgcn_cvt_off_f32_i4(w >> (8 * e + 4)));
    return r;
}

// Activations of mode M: the operand type and the exact planes that make a value.
struct Q4F16 {
    typedef _Float16 T;
    static constexpr int planes = 1, bytes = 2;
};
struct Q4BF16 {
    typedef __bf16 T;
    static constexpr int planes = 1, bytes = 2;
};
struct Q4F32 {
    typedef __bf16 T;
    static constexpr int planes = 3, bytes = 4;
};

// A workgroup takes 16 rows of a and 16 of q; its four waves share the groups of
// 128. Lane (r, h) = (l % 16, l / 16) holds weights 32 h .. + 31 of a group of row
// r, one 16-byte load; step j of the group sums k = 32 h + 8 j .. + 7. The scale
// multiplies the group's f32 sum: one a lane, as D's column is the weight row.
template <typename P>
__device__ void linear_q4(const LtxLinearQ4Args& a) {
    typedef typename P::T T;
    typedef typename Op<T>::v8 v8;
    __shared__ f32x4 part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = lane & 15, h = lane >> 4;
    const int n = blockIdx.x * 16 + r, m = blockIdx.y * 16 + r;
    const int G = a.K / LTX_GROUP;
    const uint8_t* q = a.q + (size_t)min(n, a.N - 1) * (a.K / 2) + 16 * h;
    const char* x = (const char*)a.a + ((size_t)min(m, a.M - 1) * a.K + 32 * h) * P::bytes;
    const size_t s0 = (size_t)min(n, a.N - 1) * G;
    f32x4 acc = {0, 0, 0, 0};
    for (int g = w; g < G; g += 4) {
        const u32x4 wq = *(const u32x4*)(q + 64 * (size_t)g);
        const float s = a.scale_f16 ? f16_bits_to_f32(((const uint16_t*)a.scales)[s0 + g])
                                    : ((const float*)a.scales)[s0 + g];
        f32x4 d = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const char* xp = x + ((size_t)LTX_GROUP * g + 8 * j) * P::bytes;
            const v8 wv = __builtin_bit_cast(v8, q4_operand<T>(wq[j]));
            if (P::planes == 1) {
                d = Op<T>::mfma16(__builtin_bit_cast(v8, *(const u32x4*)xp), wv, d);
            } else {
                float f[8];
                u32x4 p[3];
                *(f32x4*)f = *(const f32x4*)xp;
                *(f32x4*)(f + 4) = *(const f32x4*)(xp + 16);
                split3(f, p);
#pragma unroll
                for (int i = 0; i < 3; i++) d = Op<T>::mfma16(__builtin_bit_cast(v8, p[i]), wv, d);
            }
        }
        const float s16 = 16.0f * s;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(d[i], s16, acc[i]);
    }
    part[w][lane] = acc;
    __syncthreads();
    if (w) return;
    acc = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    if (n >= a.N) return;
    const float bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = blockIdx.y * 16 + 4 * h + i;
        if (row >= a.M) break;
        float y = acc[i] + bias;
        if (a.gelu) y = gelu_tanh(y);
        const size_t at = (size_t)row * a.N + n;
        if (a.out_f32)
            ((float*)a.y)[at] = y;
        else
            ((uint16_t*)a.y)[at] = Op<T>::bits(y);
    }
}

extern "C" __global__ void __launch_bounds__(256) ltx_linear_q4_f16(const LtxLinearQ4Args a) { linear_q4<Q4F16>(a); }
extern "C" __global__ void __launch_bounds__(256) ltx_linear_q4_bf16(const LtxLinearQ4Args a) { linear_q4<Q4BF16>(a); }
extern "C" __global__ void __launch_bounds__(256) ltx_linear_q4_f32(const LtxLinearQ4Args a) { linear_q4<Q4F32>(a); }
