// GEMMs of microscaled 4-bit operands: ltx_gemm_mx4_{f16,bf16,f32}[_gelu]_{256,128,128k2,64k2,
// 64k4,odd}, by the type of y and the tile (k2, k4: its K-tiles by groups of waves; odd:
// 128, for rows of y that do not start on 16 bytes).
#include "gemm_mx4.h"

#define MX4_GEMM_FORMS(NAME, OUT, GELU)                      \
    MX4_GEMM_KERNEL(NAME##_256, OUT, 4, GELU, true, 1, 1)    \
    MX4_GEMM_KERNEL(NAME##_128, OUT, 2, GELU, true, 1, 2)    \
    MX4_GEMM_KERNEL(NAME##_128k2, OUT, 2, GELU, true, 2, 1)  \
    MX4_GEMM_KERNEL(NAME##_64k2, OUT, 1, GELU, true, 2, 2)   \
    MX4_GEMM_KERNEL(NAME##_64k4, OUT, 1, GELU, true, 4, 1)   \
    MX4_GEMM_KERNEL(NAME##_odd, OUT, 2, GELU, false, 1, 2)
#define MX4_GEMM(TYPE, OUT)                            \
    MX4_GEMM_FORMS(ltx_gemm_mx4_##TYPE, OUT, false)    \
    MX4_GEMM_FORMS(ltx_gemm_mx4_##TYPE##_gelu, OUT, true)
MX4_GEMM(f16, _Float16)
MX4_GEMM(bf16, __bf16)
MX4_GEMM(f32, float)
