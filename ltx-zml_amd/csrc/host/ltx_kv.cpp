// The 4-bit key/value cache: its handle, rows written and read back, attention.
#include <algorithm>
#include <cstdio>
#include <cstring>

#include "ltx_internal.hpp"

struct ltx_kv_cache {
    int device = 0, mode = 0, kv_heads = 0, pages = 0;
    // blocks [pages][kv_heads], then the count of bad pages, then a flag a page
    ltx::DevBuf buf;
    size_t blocks = 0;
    // the count at the last reset: the device's is never written from here, which
    // could lose what kernels of other streams add
    unsigned long long bad_before = 0;
    uint8_t* data() const { return (uint8_t*)buf.p; }
    unsigned long long* bad() const { return (unsigned long long*)((char*)buf.p + blocks); }
    uint32_t* flags() const { return (uint32_t*)((char*)buf.p + blocks + 256); }
};

namespace ltx {
namespace {

constexpr int kMaxPages = 1 << 24; // of a table: positions stay in 31 bits

// Checks of a batch that need no device value; rows == 0 is an empty call.
LtxKvBatchArgs batch_args(const ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b) {
    if (!k || !b) throw Error("NULL argument");
    if (k->device != c->device) throw Error("the cache is on another device than the context");
    if (b->nseq <= 0 || b->rows < 0) throw Error("bad batch: nseq must be positive, rows not negative");
    if (b->max_pages <= 0 || b->max_pages > kMaxPages) throw Error("bad batch: max_pages must be 1 .. 2^24");
    if (!b->kv_len || !b->pages) throw Error("bad batch: kv_len and pages are needed");
    if (((uintptr_t)b->kv_len | (uintptr_t)b->pages | (uintptr_t)b->row_start) & 3)
        throw Error("bad batch: row_start, kv_len and pages must start on 4 bytes");
    if (!b->row_start && b->rows != b->nseq) throw Error("bad batch: without row_start, rows must equal nseq");
    return LtxKvBatchArgs{k->data(), k->flags(), k->bad(),     b->row_start, b->kv_len,
                          b->pages,  b->nseq,    b->rows, b->max_pages, k->pages, k->kv_heads};
}

void check_rows(const void* p, int64_t ld, int width, int rows, const char* what) {
    if (rows == 0) return;
    if (!p) throw Error(std::string(what) + " is NULL");
    if (ld < width || ld % 8 || ((uintptr_t)p & 15))
        throw Error(std::string(what) + ": rows must start on 16 bytes and be at least as long as their values");
}

// One launch over the rows: `write` or read.
void kv_rows(ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b, void* kp, int64_t ldk, void* vp, int64_t ldv,
             bool write, hipStream_t st) {
    LtxKvRowsArgs a{batch_args(c, k, b), kp, vp, ldk, ldv};
    const int width = k->kv_heads * LTX_HD;
    check_rows(kp, ldk, width, b->rows, "k");
    check_rows(vp, ldv, width, b->rows, "v");
    if (b->rows > (1 << 28) - 16) throw Error("too many rows for one call");  // 2^32 threads along x: one too many
    if (b->rows == 0) return;
    HIPC(hipSetDevice(c->device));
    const bool f16 = k->mode == LTX_MODE_F16;
    c->launch(write ? (f16 ? "ltx_kv_write_f16" : "ltx_kv_write_bf16") : (f16 ? "ltx_kv_read_f16" : "ltx_kv_read_bf16"),
              (unsigned)(((size_t)b->rows + 15) / 16), (k->kv_heads + 3) / 4, 1, 256, &a, st);
}

// What rows see: causal or not, and with a window the last `window` of those keys and the
// first `sinks` (window 0: none).
struct AttnMask {
    int causal = 1, window = 0, sinks = 0;
};
AttnMask mask_of(const ltx_kv_batch* b, int causal, int window, int sinks) {
    if (window < 1 || sinks < 0) throw Error("window must be positive, sinks not negative");
    const int64_t all = (int64_t)b->max_pages * LTX_KV_PAGE;  // (at most 2^30 keys)
    if (window >= all) return {causal, 0, 0};
    return {causal, window, (int)std::min<int64_t>(sinks, all)};
}
// Pages of a tile of `rows` rows, at most (the device's kv_range_units is no more).
int64_t tile_pages(const ltx_kv_batch* b, const AttnMask& m, int64_t rows) {
    if (!m.window) return b->max_pages;
    const int64_t keys = (int64_t)m.window + (m.causal ? rows + 1 : 0);
    return std::min<int64_t>(b->max_pages, ((int64_t)m.sinks + LTX_KV_PAGE - 1) / LTX_KV_PAGE +
                                               (keys + LTX_KV_PAGE - 2) / LTX_KV_PAGE + 1);
}

struct AttnPlan {
    int tile = 16;  // columns (rows times query heads of a cached head) of a tile: 16, 128 or 256
    int least = 4, slots = 0, items = 0, parts = 0;
    int64_t width = 0;  // pages of a tile, at most
    size_t bytes = 0;   // of partial results
};

// Tiles of 16 columns (eight waves that share a tile's pages), or of 128 or 256 (eight
// waves that share a page's operands). Wide tiles pay where they fill the CUs without
// a split, 256 columns before 128; a split into wide tiles only where its partial
// results (256 columns each) are spread over many pages. us on 16 / 128 / 256
// columns, `columns` a sequence:
//   one sequence of 8,192 keys, 8 cached heads: 128 columns 22 / 29 / 33, 1,024 76 /
//   82 / 77, 2,048 142 / 136 / 126, 4,096 274 / 197 / 213; of 28,672 keys: 64 columns
//   27 / 31 / 42, 256 67 / 62 / 61, 1,024 214 / 192 / 160, 4,096 808 / 674 / 565
//   32 cached heads, 2,048 keys: 512 columns 62 / 69 / 74, 1,024 114 / 56 / 112, 2,048
//   219 / 79 / 73
//   16 sequences of 2,048 keys, 8 cached heads: 64 columns 41 / 45 / 57, 128 70 / 67 /
//   75, 256 131 / 59 / 113, 512 245 / 82 / 76
//   8 sequences of 1,000 keys, 32 cached heads: 32 columns 31 / 36 / 49, 64 51 / 48 /
//   60, 128 94 / 45 / 82
// The table's width stands for the lengths, which the host does not know. A call that
// cannot split (captured, without a workspace) takes 256 columns only where they fill
// the CUs: 256 rows of 32 heads on 8 over 28,672 keys 235 us on 16 columns, 815 on 256.
// A window of few pages leaves the wide tiles' starts and ends to count, which two
// workgroups of 128 columns on a CU overlap, and the more so the more rows, each with its own
// end, a tile has. us on 128 / 256, causal, windows of 300, 1,000, 2,000 and 3,000 keys: 32
// heads on 8, 8,192 rows 97 / 107, 184 / 180, 287 / 281, 376 / 340; 32 heads, three times 4,096
// rows 165 / 225, 328 / 342, 524 / 507, 718 / 663.
// And there the 16 columns' higher cost of a page counts less than their filling of the CUs:
// about (42 + 1.9 pages) us times the share of the CUs that 128 columns would fill, those 9.5 +
// 1.4 pages. us on 16 / 128, 32 heads, windows of 300, 700, 1,400 and 2,000: 256 rows 15.5 / 15.8,
// 18 / 25, 25 / 40, 30 / 55; 512 rows 27 / 17, 32 / 25, 44 / 41, 55 / 56; 768 rows 40 / 17, 47 / 27,
// 63 / 43, 78 / 58.
int tile_columns(const ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b, const AttnMask& m, int64_t columns,
                 bool split) {
    if (c->kv_tile) return c->kv_tile;
    const int64_t group = std::max<int64_t>(1, columns / std::max(b->rows, 1));
    const int64_t each = columns / b->nseq, wide = columns * k->kv_heads / 256;  // workgroups of 256 columns
    const int64_t rows = std::min<int64_t>(256 / group, b->rows / b->nseq), width = tile_pages(b, m, rows);
    const int64_t pages = wide * width / c->num_cu;  // of each, if split
    if (each >= 192 && wide >= c->num_cu && !(m.window && width <= 12 + rows / 11)) return 256;
    if (split && each >= 256 && wide < c->num_cu && pages >= 128) return 256;
    const int64_t some = (each + 127) / 128 * b->nseq * k->kv_heads;  // workgroups of 128
    if (each >= 64 && some >= c->num_cu) return 128;
    if (m.window && each >= 128 && some * (90 + 4 * width) >= c->num_cu * (20 + 3 * width)) return 128;
    if (split && each >= 256 && wide < c->num_cu && pages >= 24) return 256;
    return 16;
}

AttnPlan attn_plan(const ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b, int heads, const AttnMask& m,
                   bool split) {
    const int64_t group = heads / k->kv_heads, columns = (int64_t)b->rows * group;
    AttnPlan p;
    p.tile = tile_columns(c, k, b, m, columns, split);
    p.width = tile_pages(b, m, p.tile / group + 1);
    // tiles of the batch, at most
    const int64_t tiles = !b->row_start || b->nseq == 1
                              ? (int64_t)b->nseq * ((columns / b->nseq + p.tile - 1) / p.tile)
                              : columns / p.tile + b->nseq;
    // the grids' limit, 2^32 threads along x; columns stay in 31 bits
    if (tiles >= (1 << 22) / k->kv_heads || columns >= 1 << 30 || b->rows >= 1 << 24)
        throw Error("too many rows for one call");
    // A split shares the pages (units, counted in 32 bits) of all tiles among one round
    // of workgroups, one a CU, and costs a launch that joins the parts: where the tiles
    // alone do not fill the CUs and are longer than 16 pages. us split / not: one row
    // of 32 cached heads, 1,000 keys 11.5 / 9.7, 2,000 11.7 / 13.0, 16,000 23 / 61; 8
    // sequences of 8 cached heads (64 workgroups), 1,000 keys 11.8 / 9.8, 4,000 20 / 21,
    // 16,000 36 / 62; of 32 (256 workgroups), 4,000 keys 32 / 29, 16,000 111 / 108;
    // ragged, 32 x 8 cached heads up to 8,192 keys 40 / 37, 8 x 32 up to 16,000 65 / 74.
    p.least = 8;
    const int64_t round = ((int64_t)c->num_cu + k->kv_heads - 1) / k->kv_heads;
    // With a window, whose range is worked out for every sequence in turn: us split / not, 32
    // cached heads, one sequence, 1,000 keys 12.1 / 10.0, 1,500 12.1 / 11.7, 2,000 12.3 / 13.3;
    // four of them, 1,000 16.3 / 10.4, 2,500 22.6 / 16.6, 4,096 24.3 / 22.4; four of 8 cached
    // heads, 2,000 15.8 / 13.4, 2,500 16.0 / 15.3, 4,096 16.1 / 20.5.
    const int64_t units = tiles * p.width, least = m.window ? 28 + (tiles - 1) * k->kv_heads * 3 / 8 : 16;
    const bool few = p.tile == 16 ? tiles * k->kv_heads < c->num_cu && p.width > least
                                  : p.tile == 256 && columns / 256 * k->kv_heads < c->num_cu && p.width > p.least;
    if (split && few && units < 1ll << 31) p.slots = (int)std::min(round, (units + p.least - 1) / p.least);
    p.items = p.slots ? p.slots : (int)tiles;
    if (p.slots) {
        p.parts = (int)(p.slots + tiles);
        p.bytes = (size_t)p.parts * k->kv_heads * p.tile * (LTX_HD + 2) * sizeof(float);
    }
    return p;
}

void check_heads(const ltx_kv_cache* k, int heads) {
    if (heads <= 0 || heads % k->kv_heads) throw Error("heads must be a positive multiple of the cache's");
    if (heads > 65535) throw Error("heads must be at most 65535");
}

// Bytes of `work`: one size serves calls with row_start and without.
uint64_t attn_workspace(const ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, int heads,
                        const AttnMask& m) {
    uint64_t bytes = attn_plan(c, cache, batch, heads, m, true).bytes;
    if (batch->rows == batch->nseq) {  // enough for the other form too: with row_start, or without
        ltx_kv_batch other = *batch;
        other.row_start = batch->row_start ? nullptr : batch->kv_len;  // (only whether there is one counts)
        try {
            bytes = std::max<uint64_t>(bytes, attn_plan(c, cache, &other, heads, m, true).bytes);
        } catch (const Error&) {  // too many rows in that form: its calls are refused
        }
    }
    return bytes;
}

struct AttnRows {
    const void* q;
    void* out;
    const float* glog;
    int64_t ldq, ldo;
    int heads;
};
void attention(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, const AttnRows& r, const AttnMask& m,
               void* work, uint64_t work_bytes, hipStream_t st) {
    LtxKvAttnArgs a{};
    a.b = batch_args(c, cache, batch);
    check_heads(cache, r.heads);
    check_rows(r.q, r.ldq, r.heads * LTX_HD, batch->rows, "q");
    check_rows(r.out, r.ldo, r.heads * LTX_HD, batch->rows, "out");
    if ((uintptr_t)r.glog & 3) throw Error("glog must start on 4 bytes");
    if ((uintptr_t)work & 15) throw Error("work must start on 16 bytes");
    AttnPlan p = attn_plan(c, cache, batch, r.heads, m, true);
    if (work && work_bytes < p.bytes) throw Error("work is smaller than the workspace call says");
    if (batch->rows == 0) return;
    HIPC(hipSetDevice(c->device));
    ScratchUse use(c->op_scratch, st);
    if (p.bytes && !work && !(work = use.take(p.bytes))) p = attn_plan(c, cache, batch, r.heads, m, false);
    a.q = r.q;
    a.out = r.out;
    a.glog = r.glog;
    a.part = (float*)work;
    a.ldq = r.ldq;
    a.ldo = r.ldo;
    a.heads = r.heads;
    a.group = r.heads / cache->kv_heads;
    a.causal = m.causal != 0;
    a.window = m.window;
    a.sinks = m.sinks;
    a.tile = p.tile;
    a.least = p.least;
    a.slots = p.slots;
    a.items = p.items;
    a.parts = p.parts;
    a.scale_log2 = 0.12751743f;  // log2(e) / sqrt(128)
    // Streaming loads where the table spans more than the memory-side cache's 256 MB
    // can help with: 499 MB (four sequences of 28,672 keys, 32 heads) 91 us against
    // 102, 557 MB 95 against 108; 278 MB, called again and again, 53 against 50
    const bool nt = (uint64_t)batch->nseq * p.width * cache->kv_heads * LTX_KV_BLOCK > 384u << 20;
    char name[48];
    auto launch = [&](const char* form, const char* end, unsigned gx, unsigned gy, unsigned threads) {
        std::snprintf(name, sizeof(name), "ltx_kv_%s_%s%s%s", form, cache->mode == LTX_MODE_F16 ? "f16" : "bf16",
                      m.window ? "_win" : "", end);
        c->launch(name, gx, gy, 1, threads, &a, st);
    };
    if (p.tile == 16)
        launch("attn", nt ? "_nt" : "", p.items, cache->kv_heads, 512);
    else
        launch("attn", p.tile == 128 ? "_rows1" : p.slots ? "_rows2_split" : "_rows2",
               (unsigned)((int64_t)p.items * cache->kv_heads), 1, 512);
    if (p.slots) launch("join", "", batch->rows, r.heads, 256);
}

}  // namespace
}  // namespace ltx

extern "C" {

int ltx_kv_cache_create(ltx_ctx* c, int mode, int kv_heads, int pages, ltx_kv_cache** out) {
    LTX_GUARD(c, {
        if (!c || !out) throw ltx::Error("NULL argument");
        *out = nullptr;
        if (mode != LTX_MODE_F16 && mode != LTX_MODE_BF16)
            throw ltx::Error("a 4-bit cache has a 16-bit mode, F16 or BF16");
        if (kv_heads <= 0 || kv_heads > 65535 || pages <= 0) throw ltx::Error("bad cache shape");
        if ((int64_t)pages * LTX_KV_PAGE > 0x7fffffff) throw ltx::Error("a cache holds at most 2^25 - 1 pages");
        HIPC(hipSetDevice(c->device));
        ltx::RelaxedCapture relaxed;
        ltx_kv_cache* k = new ltx_kv_cache();
        try {
            k->device = c->device;
            k->mode = mode;
            k->kv_heads = kv_heads;
            k->pages = pages;
            k->blocks = (size_t)pages * kv_heads * LTX_KV_BLOCK;
            k->buf.alloc(k->blocks + 256 + (size_t)pages * 4);
            // zeros: no page holds a code of a non-finite value before it is written. On a
            // stream of this call's own: a captured forward of the context has taken the
            // context's into the capture
            hipStream_t st = nullptr;
            HIPC(hipStreamCreateWithFlags(&st, hipStreamNonBlocking));
            hipError_t e = hipMemsetAsync(k->buf.p, 0, k->buf.bytes, st);
            if (e == hipSuccess) e = hipStreamSynchronize(st);
            (void)hipStreamDestroy(st);
            ltx::hip_check(e, "clearing the cache");
        } catch (...) {
            delete k;
            throw;
        }
        *out = k;
    })
}

void ltx_kv_cache_free(ltx_ctx* c, ltx_kv_cache* k) {
    if (!k) return;
    (void)c;
    (void)hipSetDevice(k->device);
    ltx::RelaxedCapture relaxed;
    delete k;  // hipFree waits for the device
}

uint64_t ltx_kv_cache_bytes(const ltx_kv_cache* k) { return k ? k->buf.bytes : 0; }

int ltx_kv_cache_faults(ltx_ctx* c, ltx_kv_cache* k, void* stream, uint64_t* count, int reset) {
    LTX_GUARD(c, {
        if (!c || !k || !count) throw ltx::Error("NULL argument");
        HIPC(hipSetDevice(c->device));
        hipStream_t st = (hipStream_t)stream;
        // (waiting for it would end the capture)
        if (ltx::is_capturing(st)) throw ltx::Error("the stream is being captured, or the legacy stream beside a capture");
        ltx::RelaxedCapture relaxed;
        unsigned long long v = 0;
        HIPC(hipMemcpyAsync(&v, k->bad(), sizeof(v), hipMemcpyDeviceToHost, st));
        HIPC(hipStreamSynchronize(st));
        *count = v - k->bad_before;
        if (reset) k->bad_before = v;
    })
}

int ltx_op_kv_write(ltx_ctx* c, ltx_kv_cache* cache, const ltx_kv_batch* batch, const void* k, int64_t ldk,
                    const void* v, int64_t ldv, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::kv_rows(c, cache, batch, (void*)k, ldk, (void*)v, ldv, true, (hipStream_t)stream);
    })
}

int ltx_op_kv_read(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, void* k, int64_t ldk, void* v,
                   int64_t ldv, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::kv_rows(c, cache, batch, k, ldk, v, ldv, false, (hipStream_t)stream);
    })
}

int ltx_op_kv_attention_workspace(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, int heads,
                                  uint64_t* bytes) {
    LTX_GUARD(c, {
        if (!c || !bytes) throw ltx::Error("NULL argument");
        ltx::batch_args(c, cache, batch);
        ltx::check_heads(cache, heads);
        *bytes = ltx::attn_workspace(c, cache, batch, heads, {});
    })
}

int ltx_op_kv_attention(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, const void* q, int64_t ldq,
                        int heads, int causal, const float* glog, void* out, int64_t ldo, void* work,
                        uint64_t work_bytes, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::attention(c, cache, batch, {q, out, glog, ldq, ldo, heads}, {causal, 0, 0}, work, work_bytes,
                       (hipStream_t)stream);
    })
}

int ltx_op_kv_attention_window_workspace(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, int heads,
                                         int causal, int window, int sinks, uint64_t* bytes) {
    LTX_GUARD(c, {
        if (!c || !bytes) throw ltx::Error("NULL argument");
        ltx::batch_args(c, cache, batch);
        ltx::check_heads(cache, heads);
        *bytes = ltx::attn_workspace(c, cache, batch, heads, ltx::mask_of(batch, causal, window, sinks));
    })
}

int ltx_op_kv_attention_window(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, const void* q,
                               int64_t ldq, int heads, int causal, int window, int sinks, const float* glog, void* out,
                               int64_t ldo, void* work, uint64_t work_bytes, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        ltx::batch_args(c, cache, batch);
        ltx::attention(c, cache, batch, {q, out, glog, ldq, ldo, heads}, ltx::mask_of(batch, causal, window, sinks),
                       work, work_bytes, (hipStream_t)stream);
    })
}

}  // extern "C"
