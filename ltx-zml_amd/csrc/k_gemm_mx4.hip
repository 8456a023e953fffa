// GEMMs of microscaled 4-bit operands: ltx_gemm_mx4_{f16,bf16}_{256,128,64}.
#include "gemm_mx4.h"

MX4_GEMM_KERNEL(ltx_gemm_mx4_f16_256, _Float16, 8, 1)
MX4_GEMM_KERNEL(ltx_gemm_mx4_bf16_256, __bf16, 8, 1)
MX4_GEMM_KERNEL(ltx_gemm_mx4_f16_128, _Float16, 4, 2)
MX4_GEMM_KERNEL(ltx_gemm_mx4_bf16_128, __bf16, 4, 2)
MX4_GEMM_KERNEL(ltx_gemm_mx4_f16_64, _Float16, 2, 2)
MX4_GEMM_KERNEL(ltx_gemm_mx4_bf16_64, __bf16, 2, 2)
