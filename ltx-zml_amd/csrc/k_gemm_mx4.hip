// GEMMs of microscaled 4-bit operands: ltx_gemm_mx4_{f16,bf16,f32}[_gelu]_{256,128,64,odd}, by
// the type of y and the tile (odd: 128, for rows of y that do not start on 16 bytes).
#include "gemm_mx4.h"

#define MX4_GEMM(TYPE, OUT)                                              \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_256, OUT, 4, false, true, 1)      \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_128, OUT, 2, false, true, 2)      \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_64, OUT, 1, false, true, 2)       \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_odd, OUT, 2, false, false, 2)     \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_256, OUT, 4, true, true, 1)  \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_128, OUT, 2, true, true, 2)  \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_64, OUT, 1, true, true, 2)   \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_odd, OUT, 2, true, false, 2)
MX4_GEMM(f16, _Float16)
MX4_GEMM(bf16, __bf16)
MX4_GEMM(f32, float)
