// A key/value cache held in 4 bits: rows written into it, read back, and
// attended to.
//
// Form. Groups of 32 dims of a row and head share a power of two 2^e, their
// values are e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6, signed). With A the
// largest magnitude of the group, e = floor(log2 A) - 2, one more where A > 7 2^e
// (what rounds past 6): 19.0 dB of signal to noise on normal values, against 18.8
// without that step. Both are limited so that 0.5 2^e and 6 2^e are finite numbers
// of the cache's 16-bit type: every code then stands for a value that type holds
// exactly, and gfx950's conversions (v_cvt_scalef32_pk_f16_fp4 and _bf16_fp4, one
// instruction a pair) give the MFMA operands without a rounding. They read only
// the scale's exponent bits, so a scale byte anywhere in a word becomes one with a
// single shift. A group that holds a non-finite value has scale code 255, which
// they turn into NaN.
#include <type_traits>

#include "ltx_device.h"
#include "ltx_kv_index.h"

template <typename T>
struct Fp4;
template <>
struct Fp4<_Float16> {
    static constexpr int lo = 127 - 23, hi = 127 + 13;
    template <int B>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, B));
    }
};
template <>
struct Fp4<__bf16> {
    static constexpr int lo = 127 - 125, hi = 127 + 125;
    template <int B>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
    }
};

// The scale whose code is byte i of w, as the conversions read it: the code at
// bits 30 .. 23 (the bits around it take no part).
__device__ __forceinline__ float scale_of(uint32_t w, int i) {
    return __builtin_bit_cast(float, i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}

// ---- the batch ----------------------------------------------------------------
// A sequence that is the same for all lanes, in scalar registers
__device__ __forceinline__ KvSeq kv_seq_all(const LtxKvBatchArgs& a, int b) {
    KvSeq s = kv_seq(a, b);
    s.s0 = __builtin_amdgcn_readfirstlane(s.s0);
    s.n = __builtin_amdgcn_readfirstlane(s.n);
    s.L = __builtin_amdgcn_readfirstlane(s.L);
    return s;
}

// The sequences of rows row0 .. row0 + 3, each lane that of row0 + sub (nseq or
// more: of none). All 64 lanes call it with one row0.
__device__ __forceinline__ int kv_find(const LtxKvBatchArgs& a, int row0, int sub) {
    if (!a.row_start) return row0 + sub;
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int base = 0; base < a.nseq; base += 64) {
        const int e = base + lane < a.nseq ? a.row_start[base + lane + 1] : 0x7fffffff;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = __popcll(__builtin_amdgcn_ballot_w64(e <= row0 + j));
            if (j == sub) b += c;
        }
    }
    return b;
}

// The first head's block of the row's page, and its key within the page; NULL where
// the row is in no sequence, before the first position, or on no page of the pool
// (`counts`: this lane counts it). in: whether it is a row of a sequence.
__device__ __forceinline__ uint8_t* kv_place(const LtxKvBatchArgs& a, int row, int b, bool counts, int& key, bool& in) {
    in = false;
    key = 0;
    if (row >= a.rows || b >= a.nseq) return nullptr;
    const KvSeq s = kv_seq(a, b);
    in = row >= s.s0 && row < s.s0 + s.n;
    const int pos = kv_position(s, row);
    if (pos < 0) return nullptr;
    const int page = kv_page(a, b, pos / LTX_KV_PAGE);
    if (!kv_in_pool(a, page)) {
        if (counts) atomicAdd(a.bad, 1ull);
        return nullptr;
    }
    key = pos % LTX_KV_PAGE;
    return a.data + kv_block(a, page, 0);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {  // over lanes 4 j .. 4 j + 3
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true));
    return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true));
}

// Eight consecutive dims of a row -> their codes, and the scale code of their
// group (four lanes hold its 32 dims).
template <typename T>
__device__ __forceinline__ uint32_t kv_encode(u32x4 w, uint32_t& code) {
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = Op<T>::to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
        top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    }
    top = quad_max(top);
    const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    code = top >= 0x7f800000u ? 255u : (uint32_t)min(max(e, Fp4<T>::lo), Fp4<T>::hi);
    const float s = __builtin_bit_cast(float, code << 23);  // (255: codes of any value)
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], s, 3);
    return q;
}

// Dword j of lane i and dword i of lane j change places, over the lanes 4 q + 0 .. 3;
__device__ __forceinline__ void quad_transpose(u32x4& x) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    auto cross = [](bool upper, uint32_t& a, uint32_t& b, auto dpp) {
        const uint32_t fa = dpp(a), fb = dpp(b);
        a = upper ? fb : a;
        b = upper ? b : fa;
    };
    uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
    auto one = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true); };
    auto two = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true); };
    cross(odd, x0, x1, one);
    cross(odd, x2, x3, one);
    cross(high, x0, x2, two);
    cross(high, x1, x3, two);
    x = u32x4{x0, x1, x2, x3};
}
// and over the lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ void row_transpose(u32x4& x) {
    auto p = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
    const uint32_t a0 = p[0], a2 = p[1];
    p = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
    const uint32_t a1 = p[0], a3 = p[1];
    p = __builtin_amdgcn_permlane16_swap(a0, a1, false, false);
    const uint32_t b0 = p[0], b1 = p[1];
    p = __builtin_amdgcn_permlane16_swap(a2, a3, false, false);
    x = u32x4{b0, b1, p[0], p[1]};
}
// x of the lane's place in its quad
__device__ __forceinline__ uint32_t quad_pick(u32x4 x) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const uint32_t low = odd ? x[1] : x[0], up = odd ? x[3] : x[2];
    return high ? up : low;
}

// Rows into the cache and out of it: a wave takes four rows of four heads, 16 lanes of
// eight dims each. Memory bounds it, and before that the count of accesses: a dword of
// codes a lane and head would be an access each. So the lanes of a quad exchange their
// K codes of four heads, and each has one head's 16 bytes; with four rows on one quad
// of positions (the rule but for a first few rows) V's codes go the same way over the
// rows, 16 bytes of four keys a lane. All of a wave's loads are on their way at once,
// and nothing here is read twice: streaming loads and stores. Measured one by one:
// 26,624 rows of 32 heads written in 137 us and read in 80 .. 91, 28,672 read in 89;
// with loads and stores that stay in the caches 164, 94 and 119 .. 152, with a dword of
// codes a lane besides 175, 185 and 213 .. 230. Back to back, where a launch waits for
// the last one's stores to reach memory, 229 for the pair and 125: 4.8 TB/s, the rate
// of a large copy.
#define KV_HB 4
template <typename T, bool WRITE>
__device__ __forceinline__ void kv_rows(const LtxKvRowsArgs& a) {
    const int lane = threadIdx.x & 63, o = lane & 15, sub = lane >> 4;
    // consecutive rows on one XCD: a page's scales are bytes of the same lines for
    // every four workgroups, and lines written in parts by several L2s are merged in
    // memory
    const uint32_t each = gridDim.x >> 3, x = blockIdx.x;
    const uint32_t group = x < 8 * each ? (x & 7) * each + (x >> 3) : x;
    const int row0 = 4 * (4 * group + (threadIdx.x >> 6)), row = row0 + sub, head0 = KV_HB * blockIdx.y;
    const int heads = min(KV_HB, a.b.kvh - head0);
    uint16_t* k = (uint16_t*)a.k + (size_t)row * a.ldk + head0 * LTX_HD + 8 * o;
    uint16_t* v = (uint16_t*)a.v + (size_t)row * a.ldv + head0 * LTX_HD + 8 * o;
    u32x4 wk[KV_HB], wv[KV_HB];
    if (WRITE)
#pragma unroll
        for (int e = 0; e < KV_HB; e++) {
            wk[e] = wv[e] = u32x4{0, 0, 0, 0};
            if (row < a.b.rows && e < heads) {
                wk[e] = __builtin_nontemporal_load((const u32x4*)(k + LTX_HD * e));
                wv[e] = __builtin_nontemporal_load((const u32x4*)(v + LTX_HD * e));
            }
        }
    const int b = kv_find(a.b, row0, sub);
    int key;
    bool in;
    uint8_t* blk = kv_place(a.b, row, b, head0 == 0 && o == 0, key, in);
    const int t = key >> 4, r = key & 15;
    // the four rows on one quad of positions
    const uint32_t place = (uint32_t)((uintptr_t)blk >> 8);  // (blocks are multiples of 256 bytes; of one pool)
    const bool together = __builtin_amdgcn_ballot_w64(
                              blk && place == (uint32_t)__builtin_amdgcn_readfirstlane((int)place) &&
                              key == (__builtin_amdgcn_readfirstlane(key) & ~3) + sub) == ~0ull;
    // what the lane holds in memory: K codes and the scales of head o % 4, V codes of
    // four keys of head sub
    const bool mine = blk && (o & 3) < heads, mine_v = sub < heads;
    uint8_t* d = blk + (size_t)(head0 + (o & 3)) * LTX_KV_BLOCK;
    uint8_t* dv = blk + (size_t)(head0 + sub) * LTX_KV_BLOCK + LTX_KV_V + 1024 * t + 16 * (16 * (r >> 2) + o);
    const uint32_t ck = 1024 * t + 256 * (o >> 2) + 16 * r;
    const uint32_t cv = LTX_KV_V + 1024 * t + 16 * (16 * (r >> 2) + o) + 4 * (r & 3);  // one key's
    const uint32_t sk = LTX_KV_KS + 64 * (o >> 2) + 4 * r + t;
    const uint32_t sv = LTX_KV_VS + 64 * (o >> 2) + 16 * (r >> 2) + 4 * t + (r & 3);
    if (WRITE) {
        u32x4 qk, qv, ek, ev;
#pragma unroll
        for (int e = 0; e < KV_HB; e++) {
            uint32_t c0, c1;
            qk[e] = kv_encode<T>(wk[e], c0);
            qv[e] = kv_encode<T>(wv[e], c1);
            ek[e] = c0;
            ev[e] = c1;
        }
        const u32x4 qv1 = qv;
        quad_transpose(qk);
        row_transpose(qv);
        const uint32_t fk = quad_pick(ek), fv = quad_pick(ev);
        if (mine) {
            *(u32x4*)(d + ck) = qk;
            d[sk] = (uint8_t)fk;
            d[sv] = (uint8_t)fv;
            if (fk == 255u || fv == 255u) a.b.flags[(size_t)(blk - a.b.data) / LTX_KV_BLOCK / a.b.kvh] = 1u;
        }
        if (together) {
            if (mine_v) *(u32x4*)dv = qv;
        } else if (blk) {
#pragma unroll
            for (int e = 0; e < KV_HB; e++)
                if (e < heads) *(uint32_t*)(blk + (size_t)(head0 + e) * LTX_KV_BLOCK + cv) = qv1[e];
        }
    } else {
        // rows of a sequence that are on no page read as zeros; rows of none stay
        u32x4 qk = {0, 0, 0, 0}, qv = {0, 0, 0, 0};
        uint32_t fk = 0, fv = 0;
        if (mine) {
            qk = *(const u32x4*)(d + ck);
            fk = d[sk];
            fv = d[sv];
        }
        if (together) {
            if (mine_v) qv = *(const u32x4*)dv;
        } else if (blk) {
#pragma unroll
            for (int e = 0; e < KV_HB; e++)
                if (e < heads) qv[e] = *(const uint32_t*)(blk + (size_t)(head0 + e) * LTX_KV_BLOCK + cv);
        }
        quad_transpose(qk);
        if (together) row_transpose(qv);
        const uint32_t sks[4] = {(uint32_t)__builtin_amdgcn_mov_dpp((int)fk, 0x00, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fk, 0x55, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fk, 0xAA, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fk, 0xFF, 0xf, 0xf, true)};
        const uint32_t svs[4] = {(uint32_t)__builtin_amdgcn_mov_dpp((int)fv, 0x00, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fv, 0x55, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fv, 0xAA, 0xf, 0xf, true),
                                 (uint32_t)__builtin_amdgcn_mov_dpp((int)fv, 0xFF, 0xf, 0xf, true)};
#pragma unroll
        for (int e = 0; e < KV_HB; e++) {
            if (!in || e >= heads) continue;
            const float sk1 = scale_of(sks[e], 0), sv1 = scale_of(svs[e], 0);
            const uint32_t q0 = qk[e], q1 = qv[e];
            const u32x4 xk = {Fp4<T>::template pair<0>(q0, sk1), Fp4<T>::template pair<1>(q0, sk1),
                              Fp4<T>::template pair<2>(q0, sk1), Fp4<T>::template pair<3>(q0, sk1)};
            const u32x4 xv = {Fp4<T>::template pair<0>(q1, sv1), Fp4<T>::template pair<1>(q1, sv1),
                              Fp4<T>::template pair<2>(q1, sv1), Fp4<T>::template pair<3>(q1, sv1)};
            __builtin_nontemporal_store(xk, (u32x4*)(k + LTX_HD * e));
            __builtin_nontemporal_store(xv, (u32x4*)(v + LTX_HD * e));
        }
    }
}

#define KV_ROWS(NAME, T, WRITE) \
    extern "C" __global__ void __launch_bounds__(256) NAME(const LtxKvRowsArgs a) { kv_rows<T, WRITE>(a); }
KV_ROWS(ltx_kv_write_f16, _Float16, true)
KV_ROWS(ltx_kv_write_bf16, __bf16, true)
KV_ROWS(ltx_kv_read_f16, _Float16, false)
KV_ROWS(ltx_kv_read_bf16, __bf16, false)

// ---- attention ------------------------------------------------------------------
// The rows of a sequence times the query heads of a cached head are its columns c =
// i * group + g; a tile is a.tile of them. Where there are few tiles, `slots` items of
// a cached head share all pages of all tiles, in order and `per` each: the k-th item
// takes units k per .. + per - 1 of them, parts of one tile or of several (a span
// each). So every item has the same work, whatever the lengths, and one round of
// workgroups does it. Each wave works the split out from the batch's arrays: lengths
// may change behind one launch (a graph's), and a table may be wider than what is in
// use. A tile that one item does whole is written by it; the partial result of item k
// for the e-th tile lies at k + e, and kv_join puts them together.
struct KvSpan {
    int b, tile, tiles;  // the tile, of the sequence's
    int page, pages;     // first unit of the span and units of the tile
    int entity;          // the tile's number in the batch
    int left;            // units left to the item
    KvSeq s;
};

__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {  // inclusive sums over the lanes
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);  // lane 15's to 16 .. 31, 47's to 48 .. 63
    x += __builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);  // lane 31's to 32 .. 63
    return x;
}

// Sequence base + lane, and what it adds to the tiles and units before the next one
struct KvLane {
    KvSeq s;
    uint32_t tiles, units, tiles_to, units_to;  // its own, and inclusive sums from `base` on
};
__device__ __forceinline__ KvLane kv_lane(const LtxKvAttnArgs& a, int base) {
    const int b = base + (threadIdx.x & 63);
    KvLane k;
    k.s = KvSeq{0, 0, 0};
    if (b < a.b.nseq) k.s = kv_seq(a.b, b);
    k.tiles = kv_tiles(k.s.n, a.group, a.tile);
    k.units = a.slots ? k.tiles * (uint32_t)kv_units(k.s.L) : k.tiles;
    k.tiles_to = wave_scan(k.tiles);
    k.units_to = wave_scan(k.units);
    return k;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int l) { return __builtin_amdgcn_readlane(x, l); }

// units an item: `first` is kv_lane(a, 0)
__device__ __forceinline__ int kv_per(const LtxKvAttnArgs& a, const KvLane& first) {
    if (!a.slots) return 1;
    uint32_t units = lane_of(first.units_to, 63);
    for (int base = 64; base < a.b.nseq; base += 64) units += lane_of(kv_lane(a, base).units_to, 63);
    return kv_per_of(units, a.slots, a.least);
}

// The item's first span; false: there is none. Without a split an item is a tile, a
// sequence's last one, which sees the most keys where the mask is causal, first.
__device__ __forceinline__ bool kv_begin(const LtxKvAttnArgs& a, int item, KvSpan& it) {
    KvLane k = kv_lane(a, 0);
    it.left = kv_per(a, k);
    const uint64_t first = (uint64_t)item * it.left;
    if (first >> 32) return false;
    uint32_t u = (uint32_t)first, entities = 0;
    for (int base = 0; base < a.b.nseq; base += 64) {
        if (base) k = kv_lane(a, base);
        const uint64_t here = __builtin_amdgcn_ballot_w64(u < k.units_to && u >= k.units_to - k.units);
        if (here) {
            const int l = __builtin_ctzll(here);
            u -= lane_of(k.units_to - k.units, l);
            it.b = base + l;
            it.s = KvSeq{(int)lane_of(k.s.s0, l), (int)lane_of(k.s.n, l), (int)lane_of(k.s.L, l)};
            it.tiles = lane_of(k.tiles, l);
            it.pages = kv_units(it.s.L);
            it.tile = a.slots ? (int)(u / (uint32_t)it.pages) : it.tiles - 1 - (int)u;
            it.page = a.slots ? (int)(u % (uint32_t)it.pages) : 0;
            it.entity = (int)(entities + lane_of(k.tiles_to - k.tiles, l)) + it.tile;
            if (!a.slots) it.left = it.pages;
            return true;
        }
        u -= lane_of(k.units_to, 63);
        entities += lane_of(k.tiles_to, 63);
    }
    return false;
}
// units of the span
__device__ __forceinline__ int kv_span(const KvSpan& it) { return min(it.left, it.pages - it.page); }
// the next one
__device__ __forceinline__ bool kv_next(const LtxKvAttnArgs& a, KvSpan& it) {
    it.left -= kv_span(it);
    if (it.left <= 0 || !a.slots) return false;
    it.page = 0;
    it.entity++;
    if (++it.tile < it.tiles) return true;
    it.tile = 0;
    while (++it.b < a.b.nseq) {
        it.s = kv_seq_all(a.b, it.b);
        it.tiles = kv_tiles(it.s.n, a.group, a.tile);
        it.pages = kv_units(it.s.L);
        if (it.tiles > 0) return true;
    }
    return false;
}

__device__ __forceinline__ float kv_quad_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// What is added to a column's sum of weights: 0, or NaN where q holds a value that is
// not finite (all of its scores are infinite or NaN then, and might all be -inf).
template <typename T>
__device__ __forceinline__ float kv_bad_query(const typename Op<T>::v8 (&q)[4]) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const u32x4 x = __builtin_bit_cast(u32x4, q[j]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t y = x[e] & 0x7fff7fffu;
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, y));
        }
    }
    const uint16_t least = __is_same(T, _Float16) ? 0x7c00 : 0x7f80;
    return top[0] >= least || top[1] >= least ? __builtin_nanf("") : 0.f;
}
// The first of sequence b's pages p0 .. p1 - 1 that is in the pool (2^24: none is).
// All 64 lanes call it.
__device__ __forceinline__ int kv_first(const LtxKvBatchArgs& a, int b, int p0, int p1) {
    for (int base = p0; base < p1; base += 64) {
        const int p = base + (threadIdx.x & 63);
        const uint64_t there = __builtin_amdgcn_ballot_w64(p < p1 && kv_in_pool(a, kv_page(a, b, p)));
        if (there) return base + __builtin_ctzll(there);
    }
    return 1 << 24;
}
// Whether a column has seen a key of pages p0 .. p1 - 1 is what its maximum says from
// here on: -inf where it has not (the mask, or pages outside the pool; its sum is 0
// then, whatever q holds), and at least -FLT_MAX where it has, also where all of its
// scores are -inf or NaN. Only a sum that is 0 or NaN leaves that open, so the table
// is looked at for such ones alone. sum: over the column's four lanes; `mine`: the keys
// that the column's mask leaves. All 64 lanes call it.
__device__ __forceinline__ void kv_seen(const LtxKvBatchArgs& a, int b, int p0, int p1, int mine, float& m, float& sum) {
    if (__builtin_amdgcn_ballot_w64(!(sum > 0.f)) == 0) return;
    const bool saw = kv_first(a, b, p0, p1) * LTX_KV_PAGE < mine;
    m = saw ? fmaxf(m, -__FLT_MAX__) : -__builtin_inff();
    sum = saw ? sum : 0.f;
}
// What a column's sums are multiplied by: 0 where it has seen no key; a sum of 0 where
// it has gives NaN (0 times infinity).
__device__ __forceinline__ float kv_factor(float m, float lt, float g) { return m == -__builtin_inff() ? 0.f : g / lt; }

// x where m is 0, y where it is ~0 (bit operations: as compares and selects, the
// rare paths below took more scalar registers than there are, in the page loop)
__device__ __forceinline__ float kv_select(int m, float x, uint32_t y) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & ~(uint32_t)m) | (y & (uint32_t)m));
}

// The scores of page p's keys that column limits leave out: -inf. s[t][i] is key 16 t
// + 4 h + i; a column sees the keys below `mine`.
__device__ __forceinline__ void kv_mask(f32x4 (&s)[4], int p, int mine, int h) {
    const int left = mine - p * LTX_KV_PAGE - 4 * h;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = kv_select((left - (16 * t + i + 1)) >> 31, s[t][i], 0xff800000u);
}

// Weights are formed and summed times 2^this (a factor that the division by their sum
// takes out again): f16's smallest number is then 2^-31 of the weight of a column's
// maximum, not 2^-24, and a maximum that is behind by 2^8 still leaves them below its
// largest. At 200,000 keys of weight 2^-25 nothing of them was left without.
template <typename T>
constexpr float kv_up = __is_same(T, _Float16) ? 7.f : 0.f;

// Online softmax of a page for a column: its scores -> weights (16-bit pairs), moved
// maximum, sum of the rounded weights. The weights are rounded to the cache's 16-bit type
// because the matrix instructions take them so; with f32 weights, as two planes, V's half
// of the products would be done twice. It costs 1.9e-4 of the result in f16 and 1.3e-3 in
// bf16 (relative RMS), beside 2.1e-4 and 1.6e-3 of the output's own rounding; the sum is of
// the rounded ones, so that equal values of V come back as they are. True: some column's maximum moved, and its
// sums are to be multiplied by corr.
template <typename T>
__device__ __forceinline__ bool kv_softmax(const f32x4 (&s)[4], float C, float& m, float& l, uint32_t (&pw)[4][2],
                                           float& corr) {
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
    mx = kv_quad_max(mx) * C;
    // a maximum that is behind by up to 2^8 stays: weights up to 256
    const bool moved = __builtin_amdgcn_ballot_w64(mx > m + 8.0f) != 0;
    if (moved) {
        const float mn = fmaxf(m, mx);
        corr = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= corr;
    }
    const float mz = (m == -__builtin_inff() ? 0.f : m) - kv_up<T>;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], C, -mz));
        // the sum takes the rounded weights, as the products do
        pw[t][0] = Op<T>::cvt2(e[0], e[1]);
        pw[t][1] = Op<T>::cvt2(e[2], e[3]);
        l = Op<T>::sum2(pw[t][1], Op<T>::sum2(pw[t][0], l));
    }
    return moved;
}

// Values of V that are not finite, in a page that has held one: a bit for each of the
// lane's 16 scales (key 16 t + 4 h + i: 4 t + i) and zeros in their place; then over
// the four groups of dims.
__device__ __forceinline__ uint32_t kv_drop_nan(u32x4& vs) {
    uint32_t bits = 0;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t y = ~vs[t];
        const uint32_t z = ~(((y & 0x7f7f7f7fu) + 0x7f7f7f7fu) | y | 0x7f7f7f7fu);  // 128 in the bytes that were 255
        vs[t] &= ~((z >> 7) * 255u);
        bits |= ((z >> 7 & 1u) | (z >> 14 & 2u) | (z >> 21 & 4u) | (z >> 28 & 8u)) << (4 * t);
    }
    bits |= __shfl_xor(bits, 4, 64);
    return bits | __shfl_xor(bits, 8, 64);
}
// The scores of those keys become NaN: a row that sees such a key is NaN, one that
// does not is untouched.
__device__ __forceinline__ void kv_set_nan(f32x4 (&s)[4], uint32_t bits) {
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = kv_select((int)(bits << (31 - 4 * t - i)) >> 31, s[t][i], 0x7fc00000u);
}

// Byte B of the codes of eight keys (x[e] of key e) with their scales -> the MFMA
// operands of its two dims.
template <typename T, int B>
__device__ __forceinline__ void kv_v_pair(const uint32_t (&x)[8], const uint32_t (&vs)[2], u32x4& lo, u32x4& hi) {
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = Fp4<T>::template pair<B>(x[e], scale_of(vs[e >> 2], e & 3));
#pragma unroll
    for (int e = 0; e < 4; e++) {
        lo[e] = __builtin_amdgcn_perm(y[2 * e + 1], y[2 * e], 0x05040100u);
        hi[e] = __builtin_amdgcn_perm(y[2 * e + 1], y[2 * e], 0x07060302u);
    }
}

#define KV_TILE 16
#define KV_WAVES 8  // (the lines below that take the waves' sums apart count on 512 threads)

// Few columns: a workgroup takes 16 columns and a run of pages, a page a wave in
// turn, everything in registers (in f16 all 256; three more values a lane wait in scratch
// while the page loop runs, which does not touch them). Scores transposed, S^T = K . Q^T, and O^T = V^T .
// P^T (v_mfma_f32_16x16x32), so that a column's statistics lie in the four lanes
// l % 16 + 16 j and P^T comes straight from the S^T accumulators. The orders in
// which dims and keys are summed are free: lane (r, h) = (l % 16, l / 16) holds
// dims 32 h .. + 31 of key 16 t + r (one 16-byte load and one scale), and for V dims
// 8 r .. + 7 of the keys 16 t + 4 h + i that its scores belong to, 16 scales in one
// load. MFMA db of O^T has dim 8 r + db in row r. All loads are contiguous over the
// lanes.
// A wave's next page is on its way while it computes on one, its index read a page
// earlier still.
// Bound: the cache's bytes. Four sequences of 28,672 keys and 32 heads (499 MB) in 87
// us, 5.7 TB/s; 32 ragged ones of up to 8,192 keys and 8 heads (146 MB, of which the
// memory-side cache holds much between calls) in 36. One short sequence is latency: a
// page's index, its codes, two rounds of products and the waves' join, 8 us.
// NT: the codes as streaming loads, for caches beyond what the memory-side cache holds.
template <typename T, bool NT>
__device__ __forceinline__ void kv_attn(const LtxKvAttnArgs& a) {
    typedef typename Op<T>::v8 v8;
    __shared__ __attribute__((aligned(16))) float so[KV_WAVES][KV_TILE][LTX_HD + 4];
    __shared__ float sm[KV_WAVES][KV_TILE], sl[KV_WAVES][KV_TILE];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = blockIdx.y;
    const float C = a.scale_log2;
    // (the constant address space: scalar loads; nothing writes them while this runs)
    typedef const __attribute__((address_space(4))) uint32_t* scalar_ptr;
    const scalar_ptr flags = (scalar_ptr)(uintptr_t)a.b.flags;
    KvSpan it;
    if (!kv_begin(a, blockIdx.x, it)) return;
    do {
        const int limit = kv_tile_limit(a.causal, it.s, a.group, it.tile, KV_TILE), np = kv_pages(limit);
        const int p0 = it.page, units = kv_span(it), p1 = min(np, p0 + units);
        const scalar_ptr table = (scalar_ptr)(uintptr_t)(a.b.pages + (size_t)it.b * a.b.max_pages);
        uint32_t next = p0 + w < p1 ? table[p0 + w] : 0u;

        // this lane's column: row, query head, keys it sees
        const int ncol = it.s.n * a.group, c0 = it.tile * KV_TILE;
        const int cols = min(KV_TILE, ncol - c0), c = min(c0 + r, ncol - 1);
        const int row = c / a.group, head = kh * a.group + c % a.group;
        const int mine = kv_limit(a.causal, it.s, row);
        const int all = kv_limit(a.causal, it.s, c0 / a.group);  // keys that every column sees
        v8 qf[4];
        const uint16_t* Q = (const uint16_t*)a.q + (size_t)(it.s.s0 + row) * a.ldq + (size_t)head * LTX_HD + 32 * h;
#pragma unroll
        for (int j = 0; j < 4; j++) qf[j] = __builtin_bit_cast(v8, *(const u32x4*)(Q + 8 * j));

        f32x4 o[8];
#pragma unroll
        for (int db = 0; db < 8; db++) o[db] = f32x4{0};
        float m = -__builtin_inff(), l = 0.f;
        struct Page {
            u32x4 k[4], v[4], vs;
            uint32_t ks, flag;
            bool none;
        };
        auto codes = [](const uint8_t* at) {
            return NT ? __builtin_nontemporal_load((const u32x4*)at) : *(const u32x4*)at;
        };
        auto load = [&](Page& x, int p) {
            if (p >= p1) return;
            x.none = next >= (uint32_t)a.b.pool;
            const uint32_t page = x.none ? 0u : next;
            // a page outside the pool: its keys are left out
            if (x.none && lane == 0 && kh == 0) atomicAdd(a.b.bad, 1ull);
            const uint8_t* blk = a.b.data + kv_block(a.b, page, kh);
            x.flag = flags[page];
#pragma unroll
            for (int t = 0; t < 4; t++) x.k[t] = codes(blk + 1024 * t + 16 * lane);
            x.ks = *(const uint32_t*)(blk + LTX_KV_KS + 4 * lane);
#pragma unroll
            for (int t = 0; t < 4; t++)
                x.v[t] = codes(blk + LTX_KV_V + 1024 * t + 16 * lane);
            x.vs = *(const u32x4*)(blk + LTX_KV_VS + 64 * (r >> 2) + 16 * h);
            next = p + KV_WAVES < p1 ? table[p + KV_WAVES] : 0u;
            __builtin_amdgcn_sched_barrier(0);
        };
        auto compute = [&](Page& x, int p) {
            f32x4 s[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float f = scale_of(x.ks, t);
                s[t] = f32x4{0};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t y = x.k[t][j];
                    const u32x4 d = {Fp4<T>::template pair<0>(y, f), Fp4<T>::template pair<1>(y, f),
                                     Fp4<T>::template pair<2>(y, f), Fp4<T>::template pair<3>(y, f)};
                    s[t] = Op<T>::mfma16(__builtin_bit_cast(v8, d), qf[j], s[t]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (x.flag) kv_set_nan(s, kv_drop_nan(x.vs));
            if (x.none || (p + 1) * LTX_KV_PAGE > all) kv_mask(s, p, x.none ? 0 : mine, h);
            uint32_t pw[4][2];
            float corr;
            if (kv_softmax<T>(s, C, m, l, pw, corr))
#pragma unroll
                for (int db = 0; db < 8; db++) o[db] *= corr;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int cc = 0; cc < 2; cc++) {
                const v8 pf = __builtin_bit_cast(v8, (u32x4){pw[2 * cc][0], pw[2 * cc][1], pw[2 * cc + 1][0],
                                                             pw[2 * cc + 1][1]});
                uint32_t y[8], f[2] = {x.vs[2 * cc], x.vs[2 * cc + 1]};
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = x.v[2 * cc + (e >> 2)][e & 3];
                auto two = [&](auto B) {  // dims 8 r + 2 B and + 1: eight keys each
                    constexpr int b = decltype(B)::value;
                    u32x4 lo, hi;
                    kv_v_pair<T, b>(y, f, lo, hi);
                    o[2 * b] = Op<T>::mfma16(__builtin_bit_cast(v8, lo), pf, o[2 * b]);
                    o[2 * b + 1] = Op<T>::mfma16(__builtin_bit_cast(v8, hi), pf, o[2 * b + 1]);
                };
                two(std::integral_constant<int, 0>{});
                two(std::integral_constant<int, 1>{});
                two(std::integral_constant<int, 2>{});
                two(std::integral_constant<int, 3>{});
            }
        };
        Page x[2];
        load(x[0], p0 + w);
#pragma nounroll
        for (int p = p0 + w; p < p1; p += 2 * KV_WAVES) {
            load(x[1], p + KV_WAVES);
            compute(x[0], p);
            if (p + KV_WAVES >= p1) break;
            load(x[0], p + 2 * KV_WAVES);
            compute(x[1], p + KV_WAVES);
        }

        // the waves' results into one: lane (r, h) holds dims 8 (4 h + i) + db
        if (p0 + w < p1) {
            l += kv_bad_query<T>(qf);
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            kv_seen(a.b, it.b, p0, p1, mine, m, l);
        }
        if (h == 0) {
            sm[w][r] = m;
            sl[w][r] = l;
        }
        if (r < cols)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float* d = &so[w][r][8 * (4 * h + i)];
                *(f32x4*)d = f32x4{o[0][i], o[1][i], o[2][i], o[3][i]};
                *(f32x4*)(d + 4) = f32x4{o[4][i], o[5][i], o[6][i], o[7][i]};
            }
        __syncthreads();
        const int col = tid >> 5, d0 = 4 * (tid & 31);
        if (col < cols) {
            float M = sm[0][col];
#pragma unroll
            for (int j = 1; j < KV_WAVES; j++) M = fmaxf(M, sm[j][col]);
            const float Mz = M == -__builtin_inff() ? 0.f : M;
            float lt = 0.f, y[4] = {};
#pragma unroll
            for (int j = 0; j < KV_WAVES; j++) {
                const float f = __builtin_amdgcn_exp2f(sm[j][col] - Mz);
                lt = __builtin_fmaf(sl[j][col], f, lt);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(so[j][col][d0 + e], f, y[e]);
            }
            const int cc = c0 + col, orow = cc / a.group, ohead = kh * a.group + cc % a.group;
            if (units < it.pages) {
                const size_t part = (size_t)blockIdx.x + it.entity, at = (part * a.b.kvh + kh) * KV_TILE + col;
                if (part < (size_t)a.parts) {
                    float* po = a.part + 2 * (size_t)a.parts * a.b.kvh * KV_TILE + at * LTX_HD + d0;
                    if (d0 == 0) *(f32x2*)(a.part + 2 * at) = f32x2{M, lt};
                    *(f32x4*)po = f32x4{y[0], y[1], y[2], y[3]};
                }
            } else {
                const int grow = it.s.s0 + orow;
                const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)grow * a.heads + ohead]) : 1.0f;
                const float f = kv_factor(M, lt, g);
                *(u32x2*)((uint16_t*)a.out + (size_t)grow * a.ldo + (size_t)ohead * LTX_HD + d0) =
                    u32x2{Op<T>::cvt2(y[0] * f, y[1] * f), Op<T>::cvt2(y[2] * f, y[3] * f)};
            }
        }
        __syncthreads();
    } while (kv_next(a, it));
}

#define KV_ATTN(NAME, T, NT)                                                                  \
    extern "C" __global__ void __launch_bounds__(64 * KV_WAVES) NAME(const LtxKvAttnArgs a) { \
        kv_attn<T, NT>(a);                                                                    \
    }
KV_ATTN(ltx_kv_attn_f16, _Float16, false)
KV_ATTN(ltx_kv_attn_bf16, __bf16, false)
KV_ATTN(ltx_kv_attn_f16_nt, _Float16, true)
KV_ATTN(ltx_kv_attn_bf16_nt, __bf16, true)

// Many columns: a workgroup takes 128 NQ columns, its eight waves 16 NQ each, and a
// run of pages. A page's codes become MFMA operands once for all eight waves, in LDS,
// in the order the operands are read (16 bytes a lane, no conflicts): waves 0 .. 3 a
// 16-key block of K each, waves 4 .. 7 half the dims of 32 keys of V each, one page
// ahead, from codes loaded two pages ahead. Two barriers a page, see below.
// Bound: a group's products of a page are 1,024 cycles of a SIMD's MFMAs and take
// about 2,200 beside the other group's exponentials and conversions and the operands'
// reads from LDS. 2,048 columns of 32 heads over 28,672 keys (962
// GFLOP) take 825 us, 1.17 PFLOP/s, causal runs of three sequences of up to 2,970
// tokens (154 GFLOP) 190. On the way there, the same call: every wave forming its own
// operands 1,675 us, operands in LDS 1,176, two groups a phase apart 1,137, loads
// without branches 1,100, one straight block of products without spills 900, staging
// before the softmax 840.
template <typename T, int NQ, bool SPLIT>
__device__ __forceinline__ void kv_attn_rows(const LtxKvAttnArgs& a) {
    typedef typename Op<T>::v8 v8;
    __shared__ __attribute__((aligned(1024))) uint8_t sk[2][16384];
    __shared__ __attribute__((aligned(1024))) uint8_t sv[2][16384];
    __shared__ uint32_t snan[2][2][4];
    // (the lane is taken anew where it is needed: what would be derived from it once
    // and kept through the loop cost more registers than there are)
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto my_lane = []() { return opaque_tid() & 63; };
    // The heads of an item follow each other, so that the large items of all heads come
    // first; where a multiple of 8 of them is cached, a head stays on one XCD. Causal,
    // 4,096 tokens: 4 cached heads 150 us against 205 with the items of a head one after
    // the other over the XCDs, 32 heads 155 against 233.
    const int item = blockIdx.x / a.b.kvh, kh = blockIdx.x - item * a.b.kvh;
    KvSpan it;
    if (!kv_begin(a, item, it)) return;
    do {
        const int limit = kv_tile_limit(a.causal, it.s, a.group, it.tile, a.tile), np = kv_pages(limit);
        const int p0 = SPLIT ? it.page : 0, units = SPLIT ? kv_span(it) : np, p1 = min(np, p0 + units);

        const int ncol = it.s.n * a.group, c0 = it.tile * a.tile + 16 * NQ * w;  // the wave's first column
        const bool idle = c0 >= ncol;
        // keys that the lane's column of block q sees
        auto limit_of = [&](int q) {
            return kv_limit(a.causal, it.s, min(c0 + 16 * q + (my_lane() & 15), ncol - 1) / a.group);
        };
        v8 qf[NQ][4];
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int lane = my_lane(), r = lane & 15, h = lane >> 4;
            const int c = min(c0 + 16 * q + r, ncol - 1), row = c / a.group;
            const uint16_t* Q = (const uint16_t*)a.q + (size_t)(it.s.s0 + row) * a.ldq +
                                (size_t)(kh * a.group + c % a.group) * LTX_HD + 32 * h;
#pragma unroll
            for (int j = 0; j < 4; j++) qf[q][j] = __builtin_bit_cast(v8, *(const u32x4*)(Q + 8 * j));
        }
        const int all = kv_limit(a.causal, it.s, min(c0, ncol - 1) / a.group);  // keys that every column sees

        // Staging. A page's index is read two pages before its codes are used, its flag
        // beside them, by scalar loads (the constant address space: nothing writes them
        // while the kernel runs); K's waves use x0 and y0. One set of loads for both kinds
        // of wave: a branch's own would be waited for where the branches meet.
        typedef const __attribute__((address_space(4))) uint32_t* scalar_ptr;
        const scalar_ptr table = (scalar_ptr)(uintptr_t)(a.b.pages + (size_t)it.b * a.b.max_pages);
        const scalar_ptr flags = (scalar_ptr)(uintptr_t)a.b.flags;
        uint32_t next = p0 < p1 ? table[p0] : 0u;  // index of the page whose codes come next
        u32x4 x0, x1;                              // its codes and scales
        uint32_t y0, y1, flag = 0, none = 0;       // its flag, or that it is outside the pool
        uint32_t flag_s = 0, none_s = 0;           // those of the page in LDS
        const int vt = 2 * ((w - 4) >> 1);         // V: first 16-key block of the wave's 32 keys
        const uint32_t ox = w < 4 ? 1024 * w : LTX_KV_V + 1024 * vt, dx = w < 4 ? 0 : 1024;
        const uint32_t oy = w < 4 ? LTX_KV_KS : LTX_KV_VS + 4 * vt, is_k = w < 4 ? ~0u : 0u;
        auto load = [&](int p) {
            none = next < (uint32_t)a.b.pool ? 0u : 1u;
            const uint32_t page = none ? 0u : next, lane = my_lane();
            if (none && w == 0 && kh == 0 && lane == 0) atomicAdd(a.b.bad, 1ull);
            const uint8_t* blk = a.b.data + kv_block(a.b, page, kh);
            x0 = *(const u32x4*)(blk + ox + 16 * lane);
            x1 = *(const u32x4*)(blk + ox + dx + 16 * lane);
            const uint32_t at = oy + (((4 * lane) & is_k) | (((lane & 12) << 4 | (lane & 48)) & ~is_k));
            y0 = *(const uint32_t*)(blk + at);
            y1 = *(const uint32_t*)(blk + at + 4);
            flag = flags[page];
            next = p + 1 < p1 ? table[p + 1] : 0u;
        };
        auto stage = [&](int buf) {
            const int lane = my_lane();
            if (w < 4) {
                const float f = __builtin_bit_cast(float, ((y0 >> (8 * w)) & 255u) << 23);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    *(u32x4*)(sk[buf] + 1024 * (4 * w + j) + 16 * lane) =
                        u32x4{Fp4<T>::template pair<0>(x0[j], f), Fp4<T>::template pair<1>(x0[j], f),
                              Fp4<T>::template pair<2>(x0[j], f), Fp4<T>::template pair<3>(x0[j], f)};
            } else {
                if (flag) {
                    u32x4 vs = {y0, y1, 0, 0};
                    const uint32_t bits = kv_drop_nan(vs);
                    y0 = vs[0];
                    y1 = vs[1];
                    if ((w & 1) == 0 && (lane & 15) == 0) snan[buf][vt >> 1][lane >> 4] = bits;
                }
                const uint32_t x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]}, f[2] = {y0, y1};
                uint8_t* d = sv[buf] + 1024 * (4 * vt) + 16 * lane;
                u32x4 lo, hi;
                if ((w & 1) == 0) {
                    kv_v_pair<T, 0>(x, f, lo, hi);
                    *(u32x4*)d = lo;
                    *(u32x4*)(d + 1024) = hi;
                    kv_v_pair<T, 1>(x, f, lo, hi);
                    *(u32x4*)(d + 2 * 1024) = lo;
                    *(u32x4*)(d + 3 * 1024) = hi;
                } else {
                    kv_v_pair<T, 2>(x, f, lo, hi);
                    *(u32x4*)(d + 4096) = lo;
                    *(u32x4*)(d + 5120) = hi;
                    kv_v_pair<T, 3>(x, f, lo, hi);
                    *(u32x4*)(d + 6144) = lo;
                    *(u32x4*)(d + 7168) = hi;
                }
            }
        };

        f32x4 o[8][NQ], s[NQ][4];  // O^T, S^T
        v8 pf[NQ][2];
        float m[NQ], l[NQ];  // running maximum (times C) and sum
#pragma unroll
        for (int q = 0; q < NQ; q++) {
#pragma unroll
            for (int db = 0; db < 8; db++) o[db][q] = f32x4{0};
            m[q] = -__builtin_inff();
            l[q] = 0.f;
        }
        const float C = a.scale_log2;
        const int nt = max(p1 - p0, 0);

        auto sync = [&]() {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        auto pv = [&](int t) {
            const uint8_t* b = sv[t & 1] + 16 * my_lane();
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int db = 0; db < 8; db++) {
                    const v8 vf = __builtin_bit_cast(v8, *(const u32x4*)(b + 1024 * (8 * c + db)));
#pragma unroll
                    for (int q = 0; q < NQ; q++) o[db][q] = Op<T>::mfma16(vf, pf[q][c], o[db][q]);
                }
        };
        auto scores = [&](int t) {
            const uint8_t* b = sk[t & 1] + 16 * my_lane();
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const v8 kf = __builtin_bit_cast(v8, *(const u32x4*)(b + 1024 * (4 * x + j)));
#pragma unroll
                    for (int q = 0; q < NQ; q++) s[q][x] = Op<T>::mfma16(kf, qf[q][j], j == 0 ? f32x4{0} : s[q][x]);
                }
        };
        // PV(t - 1), then S(t); the operands' reads run four ahead of their products
        // (masks: 0x100 DS read, 0x008 MFMA)
        auto products = [&](int t) {
            if (idle) return;
            __builtin_amdgcn_s_setprio(1);
            pv(t - 1);
            scores(t);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < 32; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, NQ, 0);
                if (i < 28) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_s_setprio(0);
        };
        // scores -> weights with maximum mc, and their sum
        auto weights = [&](int q, float mc) {
            mc -= kv_up<T>;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                u32x4 pw;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f32x4& x = s[q][2 * c + (e >> 1)];
                    const int i = 2 * (e & 1);
                    pw[e] = Op<T>::cvt2(__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], C, -mc)),
                                        __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], C, -mc)));
                    sum = Op<T>::sum2(pw[e], sum);
                }
                pf[q][c] = __builtin_bit_cast(v8, pw);
            }
            return sum;
        };
        auto softmax = [&](int t) {
            const int p = p0 + t;
            if (idle) return;
            if (flag_s) {
                const int h = my_lane() >> 4;
                const uint32_t bits = snan[t & 1][0][h] | snan[t & 1][1][h] << 8;
#pragma unroll
                for (int q = 0; q < NQ; q++) kv_set_nan(s[q], bits);
            }
            if (none_s || (p + 1) * LTX_KV_PAGE > all)
#pragma unroll
                for (int q = 0; q < NQ; q++) kv_mask(s[q], p, none_s ? 0 : limit_of(q), my_lane() >> 4);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                // weights with the maximum so far; only where a column's sum of them is
                // beyond 2^8 of it (as before it has had a score: m is -inf) the page's
                // maximum is taken, m moved, and the weights formed again
                float sum = weights(q, m[q]);
                if (__builtin_amdgcn_ballot_w64(!(sum <= (kv_up<T> ? 32768.f : 256.f))) != 0) {
                    float mx = s[q][0][0];
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[q][x][i]);
                    const float mn = fmaxf(m[q], kv_quad_max(mx) * C), mz = mn == -__builtin_inff() ? 0.f : mn;
                    const float corr = __builtin_amdgcn_exp2f(m[q] - mz);
                    m[q] = mn;
                    l[q] *= corr;
#pragma unroll
                    for (int db = 0; db < 8; db++) o[db][q] *= corr;
                    sum = weights(q, mz);
                }
                l[q] += sum;
            }
        };

        // Two groups of waves a phase apart: while one runs its products, the other runs
        // its softmax and stages (group 0 the next page's K, group 1 the next page's V),
        // so that each SIMD's matrix and vector units both have work. Phase 2 t + group:
        // products(t), phase 2 t + 1 + group: softmax(t).
        //   K(t + 1) written in phase 2 t + 1, read in 2 t + 2 and 2 t + 3; V(t + 1)
        //   written in 2 t + 2, read in 2 t + 4 and 2 t + 5; and K(t - 1)'s and V(t -
        //   1)'s buffers, which they take, were last read in 2 t - 1 and 2 t + 1.
        if (nt > 0) {
            const int group = w >> 2;
            load(p0);
            stage(0);
            flag_s = flag, none_s = none;
            if (nt > 1) load(p0 + 1);
            sync();
            if (group) sync();
            if (!idle) scores(0);
            sync();
#pragma nounroll
            for (int t = 0; t + 1 < nt; t++) {
                stage((t + 1) & 1);
                const uint32_t flag_n = flag, none_n = none;
                if (t + 2 < nt) load(p0 + t + 2);
                __builtin_amdgcn_sched_barrier(0);
                softmax(t);
                flag_s = flag_n, none_s = none_n;
                sync();
                products(t + 1);
                sync();
            }
            softmax(nt - 1);
            sync();
            if (!idle) pv(nt - 1);
            if (!group) sync();
        }

        const bool whole = !SPLIT || units == it.pages;
        const size_t part = (size_t)item + it.entity;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int lane = my_lane(), h = lane >> 4, c = c0 + 16 * q + (lane & 15);
            l[q] += kv_bad_query<T>(qf[q]);
            float lt = l[q] + __shfl_xor(l[q], 16, 64);
            lt += __shfl_xor(lt, 32, 64);
            if (!idle) kv_seen(a.b, it.b, p0, p1, limit_of(q), m[q], lt);
            if (c >= ncol || (!whole && part >= (size_t)a.parts)) continue;
            if (!whole) {
                const size_t at = (part * a.b.kvh + kh) * a.tile + (c - it.tile * a.tile);
                float* po = a.part + 2 * (size_t)a.parts * a.b.kvh * a.tile + at * LTX_HD + 32 * h;
                if (h == 0) *(f32x2*)(a.part + 2 * at) = f32x2{m[q], lt};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    *(f32x4*)(po + 8 * i) = f32x4{o[0][q][i], o[1][q][i], o[2][q][i], o[3][q][i]};
                    *(f32x4*)(po + 8 * i + 4) = f32x4{o[4][q][i], o[5][q][i], o[6][q][i], o[7][q][i]};
                }
                continue;
            }
            const int row = it.s.s0 + c / a.group, head = kh * a.group + c % a.group;
            const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)row * a.heads + head]) : 1.0f;
            const float f = kv_factor(m[q], lt, g);
            uint16_t* out = (uint16_t*)a.out + (size_t)row * a.ldo + (size_t)head * LTX_HD + 32 * h;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = Op<T>::cvt2(o[2 * e][q][i] * f, o[2 * e + 1][q][i] * f);
                *(u32x4*)(out + 8 * i) = v;
            }
        }
        if (SPLIT) __syncthreads();
    } while (SPLIT && kv_next(a, it));
}

// (the span loop costs the kernel that needs none 10 %: a kernel of its own)
#define KV_ATTN_ROWS(NAME, T, NQ, SPLIT)                                            \
    extern "C" __global__ void __launch_bounds__(512) NAME(const LtxKvAttnArgs a) { \
        kv_attn_rows<T, NQ, SPLIT>(a);                                              \
    }
KV_ATTN_ROWS(ltx_kv_attn_f16_rows1, _Float16, 1, false)
KV_ATTN_ROWS(ltx_kv_attn_bf16_rows1, __bf16, 1, false)
KV_ATTN_ROWS(ltx_kv_attn_f16_rows2, _Float16, 2, false)
KV_ATTN_ROWS(ltx_kv_attn_bf16_rows2, __bf16, 2, false)
KV_ATTN_ROWS(ltx_kv_attn_f16_rows2_split, _Float16, 2, true)
KV_ATTN_ROWS(ltx_kv_attn_bf16_rows2_split, __bf16, 2, true)

// The runs of a tile into one, where items share tiles: a workgroup takes a row and query head, a wave every
// fourth run, a lane two dims. In the runs' order: the same bits every time. Bound by
// its launch: 5 us for four rows of 32 heads.
template <typename T>
__device__ __forceinline__ void kv_join(const LtxKvAttnArgs& a) {
    __shared__ float sx[4][LTX_HD], sml[4][2];
    const int lane = threadIdx.x & 63, row = blockIdx.x, head = blockIdx.y;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the row's sequence, and the tiles and units of those before it
    KvLane k = kv_lane(a, 0);
    const int per = kv_per(a, k);
    uint32_t unit = 0, entity = 0;
    KvSeq s = {0, 0, 0};
    bool found = false;
    for (int base = 0; base < a.b.nseq; base += 64) {
        if (base) k = kv_lane(a, base);
        const uint64_t here = __builtin_amdgcn_ballot_w64(row >= k.s.s0 && row < k.s.s0 + k.s.n);
        if (here) {
            const int l = __builtin_ctzll(here);
            unit += lane_of(k.units_to - k.units, l);
            entity += lane_of(k.tiles_to - k.tiles, l);
            s = KvSeq{(int)lane_of(k.s.s0, l), (int)lane_of(k.s.n, l), (int)lane_of(k.s.L, l)};
            found = true;
            break;
        }
        unit += lane_of(k.units_to, 63);
        entity += lane_of(k.tiles_to, 63);
    }
    if (!found) return;
    const int i = row - s.s0, kh = head / a.group;
    const int c = i * a.group + head % a.group, tile = c / a.tile, col = c % a.tile, pages = kv_units(s.L);
    unit += (uint32_t)tile * pages;
    entity += tile;
    const uint32_t i0 = unit / (uint32_t)per;
    const int runs = (int)((unit + pages - 1) / (uint32_t)per - i0) + 1;
    if (runs <= 1 || (uint64_t)i0 + entity + runs > (uint64_t)a.parts) return;
    const size_t step = (size_t)a.b.kvh * a.tile, at = (((size_t)i0 + entity) * a.b.kvh + kh) * a.tile + col;
    const float* ml = a.part + 2 * at;
    const float* po = a.part + 2 * (size_t)a.parts * step + at * LTX_HD + 2 * lane;
    float M = -__builtin_inff(), lt = 0.f, x0 = 0.f, x1 = 0.f;
    for (int j0 = w; j0 < runs; j0 += 16) {  // four runs of the wave's at a time
        f32x2 v[4], y[4];
        float mn = M;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int j = min(j0 + 4 * e, runs - 1);
            v[e] = *(const f32x2*)(ml + 2 * step * j);
            y[e] = *(const f32x2*)(po + LTX_HD * step * j);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (j0 + 4 * e >= runs) v[e] = f32x2{-__builtin_inff(), 0.f};
            mn = fmaxf(mn, v[e][0]);
        }
        const float mz = mn == -__builtin_inff() ? 0.f : mn, f0 = __builtin_amdgcn_exp2f(M - mz);
        M = mn;
        lt *= f0;
        x0 *= f0;
        x1 *= f0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool there = j0 + 4 * e < runs;
            const float f = __builtin_amdgcn_exp2f(v[e][0] - mz);
            lt = there ? __builtin_fmaf(v[e][1], f, lt) : lt;
            x0 = there ? __builtin_fmaf(y[e][0], f, x0) : x0;
            x1 = there ? __builtin_fmaf(y[e][1], f, x1) : x1;
        }
    }
    *(f32x2*)&sx[w][2 * lane] = f32x2{x0, x1};
    if (lane == 0) {
        sml[w][0] = M;
        sml[w][1] = lt;
    }
    __syncthreads();
    if (w) return;
    M = fmaxf(fmaxf(sml[0][0], sml[1][0]), fmaxf(sml[2][0], sml[3][0]));
    const float Mz = M == -__builtin_inff() ? 0.f : M;
    lt = x0 = x1 = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float f = __builtin_amdgcn_exp2f(sml[j][0] - Mz);
        lt = __builtin_fmaf(sml[j][1], f, lt);
        x0 = __builtin_fmaf(sx[j][2 * lane], f, x0);
        x1 = __builtin_fmaf(sx[j][2 * lane + 1], f, x1);
    }
    const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)row * a.heads + head]) : 1.0f;
    const float f = kv_factor(M, lt, g);
    *(uint32_t*)((uint16_t*)a.out + (size_t)row * a.ldo + (size_t)head * LTX_HD + 2 * lane) =
        Op<T>::cvt2(x0 * f, x1 * f);
}

extern "C" __global__ void __launch_bounds__(256) ltx_kv_join_f16(const LtxKvAttnArgs a) { kv_join<_Float16>(a); }
extern "C" __global__ void __launch_bounds__(256) ltx_kv_join_bf16(const LtxKvAttnArgs a) { kv_join<__bf16>(a); }
