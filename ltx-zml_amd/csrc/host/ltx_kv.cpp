// The 4-bit key/value cache: its handle, rows written and read back, attention.
#include <algorithm>
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

struct AttnPlan {
    int tile = 16;  // columns (rows times query heads of a cached head) of a tile: 16, 128 or 256
    int least = 4, slots = 0, items = 0, parts = 0;
    size_t bytes = 0;  // of partial results
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
int tile_columns(const ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b, int64_t columns, bool split) {
    if (c->kv_tile) return c->kv_tile;
    const int64_t each = columns / b->nseq, wide = columns * k->kv_heads / 256;  // workgroups of 256 columns
    const int64_t pages = wide * b->max_pages / c->num_cu;                       // of each, if split
    if (each >= 192 && wide >= c->num_cu) return 256;
    if (split && each >= 256 && pages >= 128) return 256;
    if (each >= 64 && (each + 127) / 128 * b->nseq * k->kv_heads >= c->num_cu) return 128;
    if (split && each >= 256 && pages >= 24) return 256;
    return 16;
}

AttnPlan attn_plan(const ltx_ctx* c, const ltx_kv_cache* k, const ltx_kv_batch* b, int heads, bool split) {
    const int64_t group = heads / k->kv_heads, columns = (int64_t)b->rows * group;
    AttnPlan p;
    p.tile = tile_columns(c, k, b, columns, split);
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
    const int64_t units = tiles * b->max_pages;
    const bool few = p.tile == 16 ? tiles * k->kv_heads < c->num_cu && b->max_pages > 16
                                  : p.tile == 256 && columns / 256 * k->kv_heads < c->num_cu && b->max_pages > p.least;
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
        *bytes = ltx::attn_plan(c, cache, batch, heads, true).bytes;
        if (batch->rows == batch->nseq) {  // enough for the other form too: with row_start, or without
            ltx_kv_batch other = *batch;
            other.row_start = batch->row_start ? nullptr : batch->kv_len;  // (only whether there is one counts)
            try {
                *bytes = std::max<uint64_t>(*bytes, ltx::attn_plan(c, cache, &other, heads, true).bytes);
            } catch (const ltx::Error&) {  // too many rows in that form: its calls are refused
            }
        }
    })
}

int ltx_op_kv_attention(ltx_ctx* c, const ltx_kv_cache* cache, const ltx_kv_batch* batch, const void* q, int64_t ldq,
                        int heads, int causal, const float* glog, void* out, int64_t ldo, void* work,
                        uint64_t work_bytes, void* stream) {
    LTX_GUARD(c, {
        if (!c) throw ltx::Error("NULL context");
        LtxKvAttnArgs a{};
        a.b = ltx::batch_args(c, cache, batch);
        ltx::check_heads(cache, heads);
        ltx::check_rows(q, ldq, heads * LTX_HD, batch->rows, "q");
        ltx::check_rows(out, ldo, heads * LTX_HD, batch->rows, "out");
        if ((uintptr_t)glog & 3) throw ltx::Error("glog must start on 4 bytes");
        if ((uintptr_t)work & 15) throw ltx::Error("work must start on 16 bytes");
        ltx::AttnPlan p = ltx::attn_plan(c, cache, batch, heads, true);
        if (work && work_bytes < p.bytes) throw ltx::Error("work is smaller than ltx_op_kv_attention_workspace says");
        if (batch->rows == 0) return LTX_OK;
        HIPC(hipSetDevice(c->device));
        hipStream_t st = (hipStream_t)stream;
        ltx::ScratchUse use(c->op_scratch, st);
        if (p.bytes && !work && !(work = use.take(p.bytes))) p = ltx::attn_plan(c, cache, batch, heads, false);
        a.q = q;
        a.out = out;
        a.glog = glog;
        a.part = (float*)work;
        a.ldq = ldq;
        a.ldo = ldo;
        a.heads = heads;
        a.group = heads / cache->kv_heads;
        a.causal = causal != 0;
        a.tile = p.tile;
        a.least = p.least;
        a.slots = p.slots;
        a.items = p.items;
        a.parts = p.parts;
        a.scale_log2 = 0.12751743f;  // log2(e) / sqrt(128)
        const bool f16 = cache->mode == LTX_MODE_F16;
        // Streaming loads where the table spans more than the memory-side cache's 256 MB
        // can help with: 499 MB (four sequences of 28,672 keys, 32 heads) 91 us against
        // 102, 557 MB 95 against 108; 278 MB, called again and again, 53 against 50
        const bool nt = (uint64_t)batch->nseq * batch->max_pages * cache->kv_heads * LTX_KV_BLOCK > 384u << 20;
        if (p.tile == 16)
            c->launch(nt ? (f16 ? "ltx_kv_attn_f16_nt" : "ltx_kv_attn_bf16_nt") : (f16 ? "ltx_kv_attn_f16" : "ltx_kv_attn_bf16"),
                      p.items, cache->kv_heads, 1, 512, &a, st);
        else
            c->launch(p.tile == 128 ? (f16 ? "ltx_kv_attn_f16_rows1" : "ltx_kv_attn_bf16_rows1")
                      : p.slots     ? (f16 ? "ltx_kv_attn_f16_rows2_split" : "ltx_kv_attn_bf16_rows2_split")
                                    : (f16 ? "ltx_kv_attn_f16_rows2" : "ltx_kv_attn_bf16_rows2"),
                      (unsigned)((int64_t)p.items * cache->kv_heads), 1, 1, 512, &a, st);
        if (p.slots)
            c->launch(f16 ? "ltx_kv_join_f16" : "ltx_kv_join_bf16", batch->rows, heads, 1, 256, &a, st);
    })
}

}  // extern "C"
