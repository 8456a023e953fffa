// The linear with 4-bit weights.
#include <cstdio>

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
        // the grid's limits, 2^32 threads along x and 65,535 workgroups along y, and
        // 32-bit offsets of a tile's 64 rows of q and 32 of a
        if (N >= 1 << 27 || M > 65535 * 16 || K > 1 << 23) throw ltx::Error("too many rows or columns");
        HIPC(hipSetDevice(c->device));
        LtxLinearQ4Args g{a, q, scales, bias, y, M, N, K, scale_f16 != 0, gelu != 0, out_f32 != 0};
        // Tiles of 32 rows of a where there are more than 16 (mode F32: 16, its three
        // planes fill the LDS), and the fewest columns of 16, 32 or 64 whose workgroups
        // are at most one a CU: more columns a workgroup read a fewer times, fewer
        // leave no CU idle. us, 16 / 32 / 64 columns: one row of 4,096 x 4,096 5.7 / 6.8 /
        // 9.2, of 8,192 8.7 / 7.0 / 10.1, of 12,288 12.0 / 11.8 / 10.1, of 16,384 16.1 /
        // 12.4 / 10.4; 64 rows of 4,096 x 4,096 13.6 / 9.2 / 12.1, of 8,192 24.9 / 17.2 /
        // 13.4; mode F32, one row of 4,096 x 4,096 6.0 / 7.4 / 9.7, of 16,384 17.3 / 13.6 /
        // 10.9, 32 rows of 4,096 x 4,096 20.8 / 11.9 / 14.9.
        const bool f32 = mode == LTX_MODE_F32;
        const int mt = f32 || M <= 16 ? 1 : 2, gy = (M + 16 * mt - 1) / (16 * mt);
        int nt = 1;
        while (nt < 4 && ((int64_t)N + 16 * nt - 1) / (16 * nt) * gy > c->num_cu) nt *= 2;
        char name[48];
        const char* form = f32 ? M <= LTX_Q4_PACKED ? "f32p" : "f32" : mode == LTX_MODE_F16 ? "f16" : "bf16";
        std::snprintf(name, sizeof(name), "ltx_linear_q4_%s_s%d_%d_%d", form, scale_f16 ? 16 : 32, mt, nt);
        c->launch(name, (unsigned)(((int64_t)N + 16 * nt - 1) / (16 * nt)), gy, 1, 512, &g, (hipStream_t)stream);
    })
}
