// The 4-bit form of the key/value cache and of the microscaled linears: groups of 32
// values share a power of two 2^e and are held as e2m1 numbers (0, 0.5, 1, 1.5, 2, 3,
// 4, 6, signed). With A the group's largest magnitude, e = floor(log2 A) - 2, one more
// where A > 7 2^e, limited to lo - 127 .. hi - 127; its code is e + 127, or 255 for a
// group with a value that is not finite.
#pragma once
#include "ltx_device.h"

template <typename T>
struct Fp4;
template <>
struct Fp4<_Float16> {
    static constexpr int lo = 127 - 23, hi = 127 + 13;
    template <int B>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, B));
    }
};
template <>
struct Fp4<__bf16> {
    static constexpr int lo = 127 - 125, hi = 127 + 125;
    template <int B>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
    }
};
template <>
struct Fp4<float> {
    static constexpr int lo = 127 - 125, hi = 127 + 125;
};

// The scale whose code is byte i of w, as the conversions read it: the code at
// bits 30 .. 23 (the bits around it take no part).
__device__ __forceinline__ float scale_of(uint32_t w, int i) {
    return __builtin_bit_cast(float, i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {  // over lanes 4 j .. 4 j + 3
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true));
    return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true));
}

// A group's scale code from the bits of its largest magnitude.
template <typename T>
__device__ __forceinline__ uint32_t fp4_code(uint32_t top) {
    const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return top >= 0x7f800000u ? 255u : (uint32_t)min(max(e, Fp4<T>::lo), Fp4<T>::hi);
}

// Eight consecutive values of a row -> their codes, and the scale code of their
// group (four lanes hold its 32 values).
template <typename T>
__device__ __forceinline__ uint32_t fp4_encode(const float (&x)[8], uint32_t& code) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    code = fp4_code<T>(quad_max(top));
    const float s = __builtin_bit_cast(float, code << 23);  // (255: codes of any value)
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], s, 3);
    return q;
}
template <typename T>
__device__ __forceinline__ uint32_t fp4_encode(u32x4 w, uint32_t& code) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = Op<T>::to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
    return fp4_encode<T>(x, code);
}

// Dword j of lane i and dword i of lane j change places, over the lanes 4 q + 0 .. 3.
__device__ __forceinline__ void quad_transpose(u32x4& x) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    auto cross = [](bool upper, uint32_t& a, uint32_t& b, auto dpp) {
        const uint32_t fa = dpp(a), fb = dpp(b);
        a = upper ? fb : a;
        b = upper ? b : fa;
    };
    uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
    auto one = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true); };
    auto two = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true); };
    cross(odd, x0, x1, one);
    cross(odd, x2, x3, one);
    cross(high, x0, x2, two);
    cross(high, x1, x3, two);
    x = u32x4{x0, x1, x2, x3};
}
// x of the lane's place in its quad
__device__ __forceinline__ uint32_t quad_pick(u32x4 x) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const uint32_t low = odd ? x[1] : x[0], up = odd ? x[3] : x[2];
    return high ? up : low;
}
