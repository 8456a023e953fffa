// Rotary positions on several axes: their plan on the device, and the norm and rotation of
// q and k. (The tables of the block forward are ltx_rope.cpp's.)
#include <cmath>
#include <cstdio>
#include <algorithm>
#include <vector>

#include "ltx_internal.hpp"

struct ltx_rope {
    int device = 0, heads = 0, axes = 0;
    ltx::DevBuf buf;  // [heads][64] frequencies and phases, f64, in quarter turns, and axes, a byte each
    size_t pairs() const { return (size_t)heads * 64; }
    const double* freq() const { return (const double*)buf.p; }
    const double* phase() const { return freq() + pairs(); }
    const uint8_t* axis() const { return (const uint8_t*)(phase() + pairs()); }
};

namespace ltx {
namespace {

ltx_rope* rope_create(ltx_ctx* c, int heads, int axes, const double* freq, const double* phase, const int32_t* axis) {
    if (heads <= 0 || heads > 65535) throw Error("bad plan: heads must be 1 .. 65,535");
    if (axes <= 0 || axes > 8) throw Error("bad plan: axes must be 1 .. 8");
    if (!freq) throw Error("bad plan: frequencies are needed");
    const size_t n = (size_t)heads * 64;
    std::vector<double> host(2 * n + n / 8);
    uint8_t* bytes = (uint8_t*)(host.data() + 2 * n);
    for (size_t i = 0; i < n; i++) {
        host[i] = freq[i] / M_PI_2;
        host[n + i] = phase ? phase[i] / M_PI_2 : 0.0;
        if (!std::isfinite(host[i]) || !std::isfinite(host[n + i])) throw Error("bad plan: frequencies and phases must be finite");
        const int x = axis ? axis[i] : 0;
        if (x < 0 || x >= axes) throw Error("bad plan: an axis outside 0 .. axes - 1");
        bytes[i] = (uint8_t)x;
    }
    HIPC(hipSetDevice(c->device));
    RelaxedCapture relaxed;
    ltx_rope* r = new ltx_rope();
    try {
        r->device = c->device;
        r->heads = heads;
        r->axes = axes;
        r->buf.alloc(host.size() * sizeof(double));
        // on a stream of this call's own: also beside a capture
        hipStream_t st = nullptr;
        HIPC(hipStreamCreateWithFlags(&st, hipStreamNonBlocking));
        hipError_t e = hipMemcpyAsync(r->buf.p, host.data(), r->buf.bytes, hipMemcpyHostToDevice, st);
        if (e == hipSuccess) e = hipStreamSynchronize(st);
        (void)hipStreamDestroy(st);
        hip_check(e, "copying the plan");
    } catch (...) {
        delete r;
        throw;
    }
    return r;
}

}  // namespace
}  // namespace ltx

extern "C" {

int ltx_rope_create(ltx_ctx* c, int heads, int axes, const double* freq, const double* phase, const int32_t* axis,
                    ltx_rope** out) {
    LTX_GUARD(c, {
        if (!c || !out) throw ltx::Error("NULL argument");
        *out = nullptr;
        *out = ltx::rope_create(c, heads, axes, freq, phase, axis);
    })
}

int ltx_rope_create_grid(ltx_ctx* c, ltx_rope** out) {
    LTX_GUARD(c, {
        if (!c || !out) throw ltx::Error("NULL argument");
        *out = nullptr;
        // slot j of the 2,048: the identity for j < 2, else frequency (j - 2) / 3 on axis
        // (j - 2) % 3 of the position's fraction of the axis' largest, mapped to -1 .. 1
        const size_t n = LTX_H * 64;
        std::vector<double> f(n), p(n);
        std::vector<int32_t> x(n);
        for (size_t j = 2; j < n; j++) {
            const int a = (int)(j - 2) % 3;
            const double w = ltx::rope_frequency((int)(j - 2) / 3);
            f[j] = 2.0 * w / ltx::kRopeMaxPos[a];
            p[j] = -w;
            x[j] = a;
        }
        *out = ltx::rope_create(c, LTX_H, 3, f.data(), p.data(), x.data());
    })
}

void ltx_rope_free(ltx_ctx* c, ltx_rope* r) {
    if (!r) return;
    (void)c;
    (void)hipSetDevice(r->device);
    ltx::RelaxedCapture relaxed;
    delete r;  // hipFree waits for the device
}

int ltx_op_qk_rope(ltx_ctx* c, const ltx_rope* r, const double* pos, int rows, const void* q, int64_t ldq,
                   const float* q_norm, void* q_out, int64_t ldqo, int heads, const void* k, int64_t ldk,
                   const float* k_norm, void* k_out, int64_t ldko, int kv_heads, float eps, int mode, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        if (!r) throw ltx::Error("NULL argument");
        if (r->device != c->device) throw ltx::Error("the plan is on another device than the context");
        if (mode != LTX_MODE_F16 && mode != LTX_MODE_BF16 && mode != LTX_MODE_F32) throw ltx::Error("unknown mode");
        if (rows < 0) throw ltx::Error("rows must not be negative");
        if (!k) kv_heads = 0;
        if (heads <= 0 || heads % r->heads || (k && (kv_heads <= 0 || kv_heads % r->heads)))
            throw ltx::Error("heads must be positive multiples of the plan's");
        if (heads > 65535 || kv_heads > 65535) throw ltx::Error("heads must be at most 65,535");
        if (rows == 0) return LTX_OK;
        if (!pos || (uintptr_t)pos & 7) throw ltx::Error("positions are needed, on 8 bytes");
        LtxRopeArgs a{};
        const int unit = mode == LTX_MODE_F32 ? 4 : 8;
        for (int m = 0; m < (k ? 2 : 1); m++) {
            const void* x = m ? k : q;
            void* y = m ? k_out : q_out;
            const int64_t lx = m ? ldk : ldq, ly = m ? ldko : ldqo;
            const float* w = m ? k_norm : q_norm;
            const int n = m ? kv_heads : heads;
            if (!x || !y) throw ltx::Error("NULL argument");
            if (lx < n * LTX_HD || lx % unit || (uintptr_t)x & 15 || ly < n * LTX_HD || ly % unit || (uintptr_t)y & 15)
                throw ltx::Error("rows must start on 16 bytes and be at least as long as their values");
            if ((uintptr_t)w & 15) throw ltx::Error("norm weights must start on 16 bytes");
            a.x[m] = x;
            a.y[m] = y;
            a.ldx[m] = lx;
            a.ldy[m] = ly;
            a.norm[m] = w;
            a.heads[m] = n;
            a.group[m] = n / r->heads;
        }
        HIPC(hipSetDevice(c->device));
        a.freq = r->freq();
        a.phase = r->phase();
        a.axis = r->axis();
        a.pos = pos;
        a.rows = rows;
        a.axes = r->axes;
        a.eps = eps;
        const int more = std::max(heads, kv_heads), fewer = std::min(heads, kv_heads);
        const bool any = more > 32 || (fewer && more % fewer);
        const bool norm = a.norm[0] || a.norm[1];
        // workgroups that are all on the card at once (three a CU), each with its share of the rows
        a.per = (int)std::max<int64_t>(1, any ? ((int64_t)rows + (1 << 23) - 1) >> 23
                                              : ((int64_t)rows + 3 * c->num_cu - 1) / (3 * c->num_cu));
        char name[32];
        std::snprintf(name, sizeof(name), "ltx_qk_rope_%s%s",
                      mode == LTX_MODE_F16 ? "f16" : mode == LTX_MODE_BF16 ? "bf16" : "f32", any ? "_any" : norm ? "_norm" : "");
        c->launch(name, (unsigned)(((int64_t)rows + a.per - 1) / a.per), 1, 1, 256, &a, (hipStream_t)stream);
    })
}

}  // extern "C"
