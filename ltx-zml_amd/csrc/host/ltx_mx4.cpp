// Microscaled 4-bit operands: rows into the form and back, and the linear of two of them.
#include <algorithm>
#include <cstdio>

#include "ltx_internal.hpp"

namespace ltx {
namespace {

constexpr int kMaxK = 1 << 23;  // 32-bit offsets of a tile's 256 rows

const char* mode_name(int mode) {
    if (mode == LTX_MODE_F16) return "f16";
    if (mode == LTX_MODE_BF16) return "bf16";
    if (mode == LTX_MODE_F32) return "f32";
    throw Error("unknown mode");
}

// 32-bit offsets of the scale words, eight groups of 128 behind the last among them
bool scales_fit(int64_t rows, int K) { return 4 * rows * (K / 128 + 8) < 1ll << 31; }

void rows_call(ltx_ctx* c, bool quantise, void* x, int64_t ldx, uint8_t* q, uint8_t* s, int rows, int K, int mode,
               hipStream_t st) {
    char name[32];
    std::snprintf(name, sizeof(name), "ltx_mx4_%s_%s", quantise ? "quantise" : "values", mode_name(mode));
    if (rows < 0 || K <= 0 || K % 128 || K > kMaxK)
        throw Error("bad shape: rows must not be negative, K a positive multiple of 128, at most 2^23");
    if (rows == 0) return;
    if (!x || !q || !s) throw Error("NULL argument");
    if ((uintptr_t)x & 15 || (uintptr_t)q & 15 || (uintptr_t)s & 3)
        throw Error("x and the codes must start on 16 bytes, the scales on 4");
    if (ldx < K || ldx % (mode == LTX_MODE_F32 ? 4 : 8))
        throw Error("rows of x must start on 16 bytes and be at least as long as their values");
    const int64_t blocks = ((int64_t)K / 128 + 3) / 4 * (((int64_t)rows + 31) / 32);
    if (!scales_fit(rows, K) || blocks >= 1 << 24) throw Error("too many rows for one call");
    HIPC(hipSetDevice(c->device));
    LtxMx4RowsArgs a{x, q, s, ldx, rows, K};
    c->launch(name, (unsigned)blocks, 1, 1, 256, &a, st);
}

}  // namespace
}  // namespace ltx

extern "C" {

int ltx_op_mx4_quantise(ltx_ctx* c, const void* x, int64_t ldx, uint8_t* q, uint8_t* scales, int rows, int K, int mode,
                        void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::rows_call(c, true, (void*)x, ldx, q, scales, rows, K, mode, (hipStream_t)stream);
    })
}

int ltx_op_mx4_values(ltx_ctx* c, const uint8_t* q, const uint8_t* scales, void* y, int64_t ldy, int rows, int K,
                      int mode, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::rows_call(c, false, y, ldy, (uint8_t*)q, (uint8_t*)scales, rows, K, mode, (hipStream_t)stream);
    })
}

int ltx_op_linear_mx4(ltx_ctx* c, const void* a, const uint8_t* a_scales, const uint8_t* q, const uint8_t* scales,
                      const float* bias, void* y, int out_f32, int M, int N, int K, int gelu, int mode, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        const char* type = ltx::mode_name(mode);
        if (M <= 0 || N <= 0 || K <= 0 || K % 128)
            throw ltx::Error("bad linear shape: M, N and K must be positive, K a multiple of 128");
        if (!a || !q || !scales || !y) throw ltx::Error("NULL argument");
        if (mode == LTX_MODE_F32 && (!out_f32 || !a_scales))
            throw ltx::Error("mode F32 has an f32 output and takes a in the 4-bit form");
        if (!a_scales && M > LTX_MX4_ROWS) throw ltx::Error("more rows of a than 64 are taken in the 4-bit form");
        if (((uintptr_t)a | (uintptr_t)q) & 15) throw ltx::Error("a and q must start on 16 bytes");
        if (((uintptr_t)a_scales | (uintptr_t)scales) & 3) throw ltx::Error("scales must start on 4 bytes");
        if ((uintptr_t)bias & 3 || (uintptr_t)y & (out_f32 ? 3 : 1))
            throw ltx::Error("bias and y must be aligned to their types");
        // (32-bit offsets of a tile's 256 rows of y)
        if (K > ltx::kMaxK || !ltx::scales_fit(M, K) || !ltx::scales_fit(N, K) || N >= 1 << 21)
            throw ltx::Error("too many rows or columns");
        HIPC(hipSetDevice(c->device));
        hipStream_t st = (hipStream_t)stream;
        if (mode == LTX_MODE_F32) type = "f16";  // (codes in, f32 out: no type takes part)
        LtxMx4LinearArgs g{};
        g.a = (const uint8_t*)a;
        g.as = a_scales;
        g.w = q;
        g.ws = scales;
        g.bias = bias;
        g.y = y;
        g.M = M;
        g.N = N;
        g.K = K;
        g.gelu = gelu != 0;
        g.out_f32 = out_f32 != 0;
        char name[48];
        const int64_t cu = c->num_cu;
        auto tiles = [&](int64_t t) { return (M + t - 1) / t * ((N + t - 1) / t); };
        if (!a_scales || (c->mx4_tile ? c->mx4_tile == 16 && M <= 1 << 20 : M <= LTX_MX4_ROWS)) {
            const int mt = std::min((M + 15) / 16, 4);
            int nt = 1;
            while (nt < (mt > 2 ? 2 : 4) && ((int64_t)N + 16 * nt - 1) / (16 * nt) > cu) nt *= 2;
            std::snprintf(name, sizeof(name), "ltx_linear_mx4_%s_%s%d_%d", type, a_scales ? "" : "rows_", mt, nt);
            c->launch(name, (unsigned)((N + 16 * nt - 1) / (16 * nt)), (unsigned)((M + 16 * mt - 1) / (16 * mt)), 1, 512, &g,
                      st);
            return LTX_OK;
        }
        const bool odd = (uintptr_t)y & 15 || N % (out_f32 ? 4 : 8);  // rows of y that do not start on 16 bytes
        const int tile = odd ? 128 : c->mx4_tile > 16 ? c->mx4_tile : tiles(256) >= cu ? 256 : tiles(128) >= cu ? 128 : 64;
        g.tiles_m = (M + tile - 1) / tile;
        g.tiles_n = (N + tile - 1) / tile;
        const int64_t n = tiles(tile);
        if (n >= 1 << 23) throw ltx::Error("too many rows or columns");  // (twice: past the last, an index stays in 31 bits)
        const char* form = odd ? "odd" : tile == 256 ? "256" : tile == 128 ? "128" : "64";
        std::snprintf(name, sizeof(name), "ltx_gemm_mx4_%s%s_%s", out_f32 ? "f32" : type, gelu ? "_gelu" : "", form);
        c->launch(name, (unsigned)(tile == 256 ? std::min(n, cu) : n), 1, 1, 256, &g, st);
    })
}

}  // extern "C"
