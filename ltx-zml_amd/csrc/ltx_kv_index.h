// Index arithmetic of the 4-bit cache and of its attention's work split, for the
// kernels and, compiled by a host compiler, for what is checked without a GPU: for
// any contents of the batch's device arrays, rows stay in 0 .. rows - 1, table
// entries in 0 .. max_pages - 1 and places in the pool.
#pragma once
#include "ltx_args.h"
#ifdef __HIPCC__
#define KV_FN __device__ __forceinline__
#else
#define KV_FN inline
#endif

KV_FN int64_t kv_min(int64_t a, int64_t b) { return a < b ? a : b; }
KV_FN int64_t kv_max(int64_t a, int64_t b) { return a > b ? a : b; }

// Sequence b: its rows s0 .. s0 + n - 1 are positions L - n .. L - 1. What the
// device arrays hold is limited to the rows and the table that the call names.
struct KvSeq {
    int s0, n, L;
};
KV_FN KvSeq kv_seq(const LtxKvBatchArgs& a, int b) {
    KvSeq s;
    int e = b + 1;
    s.s0 = b;
    if (a.row_start) {
        s.s0 = (int)kv_min(kv_max(a.row_start[b], 0), a.rows);
        e = (int)kv_min(kv_max(a.row_start[b + 1], s.s0), a.rows);
    }
    s.n = e - s.s0;
    s.L = (int)kv_min(kv_max(a.kv_len[b], 0), (int64_t)a.max_pages * LTX_KV_PAGE);
    return s;
}

// Of row `row`, a row of sequence b: its position, or -1 (no row of the sequence,
// or before the first position).
KV_FN int kv_position(const KvSeq& s, int row) {
    const int i = row - s.s0;
    if (i < 0 || i >= s.n) return -1;
    const int pos = s.L - s.n + i;
    return pos < 0 ? -1 : pos;
}
// The table's page p of sequence b; outside the pool: the caller leaves it out.
KV_FN int kv_page(const LtxKvBatchArgs& a, int b, int p) { return a.pages[(size_t)b * a.max_pages + p]; }
KV_FN bool kv_in_pool(const LtxKvBatchArgs& a, int page) { return (unsigned)page < (unsigned)a.pool; }
KV_FN size_t kv_block(const LtxKvBatchArgs& a, int page, int head) {
    return ((size_t)page * a.kvh + head) * LTX_KV_BLOCK;
}

KV_FN int kv_pages(int keys) { return (int)(((int64_t)keys + LTX_KV_PAGE - 1) / LTX_KV_PAGE); }
KV_FN int kv_tiles(int n, int group, int tile) { return (int)(((int64_t)n * group + tile - 1) / tile); }
// Work of a split attention call: a tile's pages, one at least (a tile without keys
// still writes its zeros); and the pages that each of about `slots` items takes of
// all of them.
KV_FN int kv_units(int keys) { return (int)kv_max(1, kv_pages(keys)); }
KV_FN int kv_per_of(uint32_t units, int slots, int least) {
    return (int)kv_max(least, ((int64_t)units + slots - 1) / slots);
}

// keys that row i of the sequence sees
KV_FN int kv_limit(int causal, const KvSeq& s, int i) {
    return causal ? (int)kv_max(0, (int64_t)s.L - s.n + i + 1) : s.L;
}
// and the last row of tile t
KV_FN int kv_tile_limit(int causal, const KvSeq& s, int group, int t, int tile) {
    const int64_t c = kv_min((int64_t)(t + 1) * tile, (int64_t)s.n * group) - 1;
    return kv_limit(causal, s, (int)(c / group));
}
