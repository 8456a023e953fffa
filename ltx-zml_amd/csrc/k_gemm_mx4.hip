// GEMMs of microscaled 4-bit operands: ltx_gemm_mx4_{f16,bf16,f32}[_gelu]_{256,128,64}, by
// the type of y and the tile.
#include "gemm_mx4.h"

#define MX4_GEMM(TYPE, OUT)                                                \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_256, OUT, 4, false, 1)           \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_128, OUT, 2, false, 2)           \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_64, OUT, 1, false, 2)            \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_256, OUT, 4, true, 1)       \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_128, OUT, 2, true, 2)       \
    MX4_GEMM_KERNEL(ltx_gemm_mx4_##TYPE##_gelu_64, OUT, 1, true, 2)
MX4_GEMM(f16, _Float16)
MX4_GEMM(bf16, __bf16)
MX4_GEMM(f32, float)
