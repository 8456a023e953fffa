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

// 32-bit offsets of the scale words, sixteen groups of 128 behind the last among them
bool scales_fit(int64_t rows, int K) { return 4 * rows * (K / 128 + 16) < 1ll << 31; }

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

struct Mx4Form {
    int tile, groups;  // 16: the kernel of few rows
    const char* name;
};

// Tiles of 256 x 256 where they come near to filling the CUs; of 128, two workgroups a CU; and
// where few tiles leave a K-tile's latency to count, several groups of waves on one tile. us
// at K = 4,096, few rows / 64k2 / 64k4 / 128 / 128k2 / 256:
//   M   16 x N  4,096    4.4 /  5.9 /  5.8 /  9.6 /  9.1 /   -
//       32 x    4,096    5.5 /  5.8 /  5.9 /  9.6 /  9.2 /   -
//       64 x    4,096    8.2 /  5.9 /  6.0 /  9.8 /  9.3 /   -
//       16 x    8,192    6.1 /  5.8 /  5.9 /  9.5 /  9.2 /   -
//       16 x   12,288    8.5 /  6.4 /  6.2 / 10.5 /  9.3 /   -
//      128 x   16,384   27   / 10.5 / 14.0 / 14.9 / 12.8 /   -
//      256 x   12,288    -   / 15.5 / 19.0 / 14.0 / 12.3 /   -
//      512 x    4,096    -   /  9.9 / 11.8 / 10.6 / 10.1 /   -
//      640 x   12,288    -   / 37   / 49   / 23   / 28   / 29
//    1,024 x    4,096    -   / 20   / 26   / 14.1 / 13.5 / 27
//    1,024 x   12,288    -   / 54   / 71   / 36   / 39   / 32
//    2,048 x    8,192    -   / 69   / 94   / 44   / 52   / 37
// K = 16,384, N = 4,096: 16 rows 12 / 22 / 17 / 41 / 32, 64 26 / 23 / 19 / 42 / 33, 256 - / 24 /
// 21 / 44 / 35, 512 - / 31 / 39 / 44 / 35, 2,970 - / 165 / 220 / 114 / 123 / 96; K = 1,024, 64
// rows 4.0 / 3.6 / 4.7 / 5.2 / 5.2.
// Rows of y that do not start on 16 bytes (`odd`) have one form, 128 x 128 with narrow stores,
// whatever the sizes: the others exist for whole 16-byte stores only. us at N = 4,097 / 4,104, f16:
// K = 4,096, 64 rows 12.5 / 6.3, 300 19.3 / 11.1, 2,048 56 / 34, 28,672 478 / 238; K = 16,384, 64
// rows 45 / 20, 300 51 / 30, 2,048 133 / 112.
Mx4Form mx4_form(const ltx_ctx* c, int64_t M, int64_t N, int K, bool rows, bool odd) {
    auto tiles = [&](int64_t t) { return (M + t - 1) / t * ((N + t - 1) / t); };
    const int64_t cu = c->num_cu;
    const Mx4Form few{16, 1, ""};
    if (rows || c->mx4_tile == 16 || (!c->mx4_tile && ((M <= 32 && N <= 16 * cu) || (M <= 16 && N <= 32 * cu)))) return few;
    if (odd) return {128, 1, "odd"};
    const int t = c->mx4_tile;
    if (t ? t == 64 : tiles(64) <= 2 * cu)
        return tiles(64) <= cu && K >= 4096 ? Mx4Form{64, 4, "64k4"} : Mx4Form{64, 2, "64k2"};
    if (t ? t == 128 : tiles(256) < 3 * cu / 4) return tiles(128) <= cu ? Mx4Form{128, 2, "128k2"} : Mx4Form{128, 1, "128"};
    return {256, 1, "256"};
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
        // Rows in values: up to 16, and few values, are quantised by every workgroup that
        // multiplies them, others once, by a launch of their own, into scratch (whose order
        // behind other calls takes 3 us). us, in the product / in a launch: K = 1,024, N =
        // 16,384, 17 rows 5.6 / 10.8, 64 10.8 / 11.3; K = 4,096, N = 4,096, 17 rows 8.1 / 11.9, 32
        // 10.9 / 12.6, 48 15.2 / 13.8, 64 18.7 / 14.3, and N = 16,384 12.9 / 14.9, 16.3 / 15.2, 21.0
        // / 16.5, 25.6 / 16.3; K = 16,384, N = 4,096, 17 rows 25 / 20, 64 65 / 27. (N is not in the
        // rule: its worst case among these, 32 rows of 16,384 x 4,096, is 7 % slower than a launch.)
        ltx::ScratchUse use(c->op_scratch, st);
        if (!a_scales && M > 16 && (int64_t)M * K > 1 << 17) {
            const size_t codes = (size_t)M * K / 2;
            if (uint8_t* s = (uint8_t*)use.take(codes + (size_t)M * K / 32)) {
                ltx::rows_call(c, true, (void*)a, K, s, s + codes, M, K, mode, st);
                g.a = s;
                g.as = s + codes;
            }
        }
        const ltx::Mx4Form form = ltx::mx4_form(c, M, N, K, !g.as, (uintptr_t)y & 15 || N % (out_f32 ? 4 : 8));
        char name[48];
        if (form.tile == 16) {
            const int mt = std::min((M + 15) / 16, g.as ? 2 : 4);
            // the fewest columns of 16, 32 or 64 whose workgroups are at most one a CU (codes: where
            // these kernels are taken, 16 or, up to 16 rows, 32)
            int nt = 1;
            while (nt < (!g.as ? 4 : mt == 1 ? 2 : 1) && ((int64_t)N + 16 * nt - 1) / (16 * nt) > c->num_cu) nt *= 2;
            std::snprintf(name, sizeof(name), "ltx_linear_mx4_%s_%s%d_%d", type, g.as ? "" : "rows_", mt, nt);
            c->launch(name, (unsigned)((N + 16 * nt - 1) / (16 * nt)), (unsigned)((M + 16 * mt - 1) / (16 * mt)), 1, 512, &g,
                      st);
            return LTX_OK;
        }
        g.tiles_m = (M + form.tile - 1) / form.tile;
        g.tiles_n = (N + form.tile - 1) / form.tile;
        const int64_t n = (int64_t)g.tiles_m * g.tiles_n;
        if (n >= 1 << 22) throw ltx::Error("too many rows or columns");  // (2^32 threads along x)
        std::snprintf(name, sizeof(name), "ltx_gemm_mx4_%s%s_%s", out_f32 ? "f32" : type, gelu ? "_gelu" : "", form.name);
        c->launch(name, (unsigned)(form.tile == 256 ? std::min<int64_t>(n, c->num_cu) : n), 1, 1, 256 * form.groups, &g, st);
    })
}

}  // extern "C"
