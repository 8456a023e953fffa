// The linear with 4-bit weights.
#include "ltx_internal.hpp"

extern "C" int ltx_op_linear_q4(ltx_ctx* c, const void* a, const uint8_t* q, const void* scales, int scale_f16,
                                const float* bias, void* y, int out_f32, int M, int N, int K, int gelu, int mode,
                                void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        if (mode != LTX_MODE_F16 && mode != LTX_MODE_BF16 && mode != LTX_MODE_F32) throw ltx::Error("unknown mode");
        if (M <= 0 || N <= 0 || K <= 0 || K % LTX_GROUP)
            throw ltx::Error("bad linear shape: M, N and K must be positive, K a multiple of 128");
        if (!a || !q || !scales || !y) throw ltx::Error("NULL argument");
        if (((uintptr_t)a | (uintptr_t)q) & 15) throw ltx::Error("a and q must start on 16 bytes");
        if ((uintptr_t)scales & (scale_f16 ? 1 : 3)) throw ltx::Error("scales must be aligned to their type");
        if ((uintptr_t)bias & 3 || (uintptr_t)y & (out_f32 || mode == LTX_MODE_F32 ? 3 : 1))
            throw ltx::Error("bias and y must be aligned to their types");
        if (mode == LTX_MODE_F32 && !out_f32) throw ltx::Error("mode F32 has an f32 output");
        if (((int64_t)N + 15) / 16 >= 1 << 24 || ((int64_t)M + 15) / 16 > 65535) throw ltx::Error("too many rows");
        HIPC(hipSetDevice(c->device));
        LtxLinearQ4Args g{a, q, scales, bias, y, M, N, K, scale_f16 != 0, gelu != 0, out_f32 != 0};
        c->launch(mode == LTX_MODE_F16    ? "ltx_linear_q4_f16"
                  : mode == LTX_MODE_BF16 ? "ltx_linear_q4_bf16"
                                          : "ltx_linear_q4_f32",
                  (N + 15) / 16, (M + 15) / 16, 1, 256, &g, (hipStream_t)stream);
    })
}
