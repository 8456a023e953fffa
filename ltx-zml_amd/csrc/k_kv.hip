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

// The block of (row's position, head), and its key within the page; NULL where the
// row is in no sequence, before the first position, or on no page of the pool.
__device__ __forceinline__ uint8_t* kv_place(const LtxKvBatchArgs& a, int row, int b, int head, int& key) {
    if (row >= a.rows || b >= a.nseq) return nullptr;
    const int pos = kv_position(kv_seq(a, b), row);
    if (pos < 0) return nullptr;
    const int page = kv_page(a, b, pos / LTX_KV_PAGE);
    if (!kv_in_pool(a, page)) {
        if (head == 0 && (threadIdx.x & 15) == 0) atomicAdd(a.bad, 1ull);
        return nullptr;
    }
    key = pos % LTX_KV_PAGE;
    return a.data + kv_block(a, page, head);
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
    if (code == 255u) return 0u;
    const float s = __builtin_bit_cast(float, code << 23);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], s, 3);
    return q;
}

// Rows into the cache and out of it: a wave takes four rows of a head, 16 lanes of
// eight dims each. Four positions of a quad are 256 consecutive bytes of V codes.
template <typename T, bool WRITE>
__device__ void kv_rows(const LtxKvRowsArgs& a) {
    const int lane = threadIdx.x & 63, o = lane & 15, sub = lane >> 4;
    const int row0 = 4 * (4 * blockIdx.x + (threadIdx.x >> 6)), row = row0 + sub, head = blockIdx.y;
    const int b = kv_find(a.b, row0, sub);
    int key = 0;
    uint8_t* blk = kv_place(a.b, row, b, head, key);
    const int t = key >> 4, r = key & 15;
    uint16_t* k = (uint16_t*)a.k + (size_t)row * a.ldk + head * LTX_HD + 8 * o;
    uint16_t* v = (uint16_t*)a.v + (size_t)row * a.ldv + head * LTX_HD + 8 * o;
    const uint32_t ck = 1024 * t + 256 * (o >> 2) + 16 * r + 4 * (o & 3), sk = LTX_KV_KS + 64 * (o >> 2) + 4 * r + t;
    const uint32_t cv = LTX_KV_V + 1024 * t + 16 * (16 * (r >> 2) + o) + 4 * (r & 3);
    const uint32_t sv = LTX_KV_VS + 64 * (o >> 2) + 16 * (r >> 2) + 4 * t + (r & 3);
    if (WRITE) {
        const u32x4 zero = {0, 0, 0, 0};
        const u32x4 wk = blk ? *(const u32x4*)k : zero, wv = blk ? *(const u32x4*)v : zero;
        uint32_t ek, ev;
        const uint32_t qk = kv_encode<T>(wk, ek), qv = kv_encode<T>(wv, ev);
        if (!blk) return;
        *(uint32_t*)(blk + ck) = qk;
        *(uint32_t*)(blk + cv) = qv;
        if ((o & 3) == 0) {
            blk[sk] = (uint8_t)ek;
            blk[sv] = (uint8_t)ev;
            if (ek == 255u || ev == 255u)
                a.b.flags[(size_t)(blk - a.b.data) / LTX_KV_BLOCK / a.b.kvh] = 1u;
        }
    } else {
        // rows of a sequence that are on no page read as zeros; rows of none stay
        if (row >= a.b.rows || b >= a.b.nseq) return;
        const KvSeq s = kv_seq(a.b, b);
        if (row < s.s0 || row >= s.s0 + s.n) return;
        u32x4 wk = {0, 0, 0, 0}, wv = {0, 0, 0, 0};
        if (blk) {
            const uint32_t qk = *(const uint32_t*)(blk + ck), qv = *(const uint32_t*)(blk + cv);
            const float fk = __builtin_bit_cast(float, (uint32_t)blk[sk] << 23);
            const float fv = __builtin_bit_cast(float, (uint32_t)blk[sv] << 23);
            wk = u32x4{Fp4<T>::template pair<0>(qk, fk), Fp4<T>::template pair<1>(qk, fk),
                       Fp4<T>::template pair<2>(qk, fk), Fp4<T>::template pair<3>(qk, fk)};
            wv = u32x4{Fp4<T>::template pair<0>(qv, fv), Fp4<T>::template pair<1>(qv, fv),
                       Fp4<T>::template pair<2>(qv, fv), Fp4<T>::template pair<3>(qv, fv)};
        }
        *(u32x4*)k = wk;
        *(u32x4*)v = wv;
    }
}

#define KV_ROWS(NAME, T, WRITE) \
    extern "C" __global__ void __launch_bounds__(256) NAME(const LtxKvRowsArgs a) { kv_rows<T, WRITE>(a); }
KV_ROWS(ltx_kv_write_f16, _Float16, true)
KV_ROWS(ltx_kv_write_bf16, __bf16, true)
KV_ROWS(ltx_kv_read_f16, _Float16, false)
KV_ROWS(ltx_kv_read_bf16, __bf16, false)

// ---- attention ------------------------------------------------------------------
// Items. The rows of a sequence times the query heads of a cached head are its
// columns c = i * group + g; a tile is `tile` of them. Its keys are split into runs
// of `per` pages, the same for all sequences: as many as make about `slots` items of
// a cached head in all. Every wave works the split out from the batch's lengths, so
// lengths may change behind one launch (a graph's), and a table may be wider than
// what is in use. Items: sequence by sequence, tile by tile, run by run.
struct KvItem {
    int b, tile, run;
    KvSeq s;
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
    return v;
}

// pages a run
__device__ __forceinline__ int kv_per(const LtxKvAttnArgs& a) {
    if (a.slots == 0) return KV_NO_SPLIT;
    const int lane = threadIdx.x & 63;
    uint64_t w = 0;
    if (a.b.nseq == 1) {
        const KvSeq s = kv_seq(a.b, 0);
        w = (uint64_t)kv_tiles(s.n, a.group, a.tile) * kv_pages(s.L);
    } else {
        for (int b = lane; b < a.b.nseq; b += 64) {
            const KvSeq s = kv_seq(a.b, b);
            w += (uint64_t)kv_tiles(s.n, a.group, a.tile) * kv_pages(s.L);
        }
        w = wave_sum(w);
    }
    return kv_per_of(w, a.slots, a.least);
}

// The item's sequence, tile and run; false: there is none. A sequence's last tile,
// which sees the most keys where the mask is causal, comes first.
__device__ __forceinline__ bool kv_item(const LtxKvAttnArgs& a, int per, int item, KvItem& it) {
    if (a.b.nseq == 1) {
        it.b = 0;
    } else {
        const int lane = threadIdx.x & 63;
        it.b = -1;
        for (int base = 0; base < a.b.nseq; base += 64) {
            int c = 0;
            if (base + lane < a.b.nseq) {
                const KvSeq s = kv_seq(a.b, base + lane);
                c = kv_tiles(s.n, a.group, a.tile) * kv_runs(kv_pages(s.L), per);
            }
            int sum = c;
            for (int o = 1; o < 64; o <<= 1) {
                const int up = __shfl_up(sum, o, 64);
                if (lane >= o) sum += up;
            }
            const uint64_t here = __builtin_amdgcn_ballot_w64(item < sum && item >= sum - c);
            if (here) {
                const int l = __builtin_ctzll(here);
                it.b = base + l;
                item -= __shfl(sum - c, l, 64);
                break;
            }
            item -= __shfl(sum, 63, 64);
        }
        it.b = __builtin_amdgcn_readfirstlane(it.b);
        item = __builtin_amdgcn_readfirstlane(item);
        if (it.b < 0) return false;
    }
    it.s = kv_seq(a.b, it.b);
    const int runs = kv_runs(kv_pages(it.s.L), per);
    it.tile = kv_tiles(it.s.n, a.group, a.tile) - 1 - item / runs;
    it.run = item % runs;
    return it.tile >= 0;
}

__device__ __forceinline__ float kv_quad_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// The scores of page p's keys that column limits leave out: -inf. s[t][i] is key 16 t
// + 4 h + i; a column sees the keys below `mine`.
__device__ __forceinline__ void kv_mask(f32x4 (&s)[4], int p, int mine, int h) {
    const int left = mine - p * LTX_KV_PAGE - 4 * h;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (16 * t + i >= left) s[t][i] = -__builtin_inff();
}

// Online softmax of a page for a column: its scores -> weights (16-bit pairs), moved
// maximum, sum of the rounded weights. True: some column's maximum moved, and its
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
    const float mz = m == -__builtin_inff() ? 0.f : m;
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
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (((vs[t] >> (8 * i)) & 255u) == 255u) {
                bits |= 1u << (4 * t + i);
                vs[t] &= ~(255u << (8 * i));
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
        for (int i = 0; i < 4; i++)
            if (bits & (1u << (4 * t + i))) s[t][i] = __builtin_nanf("");
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

// Few columns: a workgroup takes 16 columns and a run of pages, a page a wave in
// turn, everything in registers. Scores transposed, S^T = K . Q^T, and O^T = V^T .
// P^T (v_mfma_f32_16x16x32), so that a column's statistics lie in the four lanes
// l % 16 + 16 j and P^T comes straight from the S^T accumulators. The orders in
// which dims and keys are summed are free: lane (r, h) = (l % 16, l / 16) holds
// dims 32 h .. + 31 of key 16 t + r (one 16-byte load and one scale), and for V dims
// 8 r .. + 7 of the keys 16 t + 4 h + i that its scores belong to, 16 scales in one
// load. MFMA db of O^T has dim 8 r + db in row r. All loads are contiguous over the
// lanes.
template <typename T>
__device__ void kv_attn(const LtxKvAttnArgs& a) {
    typedef typename Op<T>::v8 v8;
    __shared__ __attribute__((aligned(16))) float so[4][KV_TILE][LTX_HD + 4];
    __shared__ float sm[4][KV_TILE], sl[4][KV_TILE];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = blockIdx.y;
    const int per = kv_per(a);
    KvItem it;
    if (!kv_item(a, per, blockIdx.x, it)) return;
    const int limit = kv_tile_limit(a.causal, it.s, a.group, it.tile, KV_TILE), np = kv_pages(limit);
    const int p0 = it.run * per, p1 = min(np, p0 + min(per, np));
    if (it.run > 0 && p0 >= np) return;

    // this lane's column: row, query head, keys it sees
    const int64_t ncol = (int64_t)it.s.n * a.group;
    const int64_t c0 = (int64_t)it.tile * KV_TILE;
    const int cols = (int)min((int64_t)KV_TILE, ncol - c0);
    const int64_t c = min(c0 + r, ncol - 1);
    const int row = (int)(c / a.group), head = kh * a.group + (int)(c % a.group);
    const int mine = kv_limit(a.causal, it.s, row);
    const int all = kv_limit(a.causal, it.s, (int)(c0 / a.group));  // keys that every column sees
    v8 qf[4];
    const uint16_t* Q = (const uint16_t*)a.q + (size_t)(it.s.s0 + row) * a.ldq + (size_t)head * LTX_HD + 32 * h;
#pragma unroll
    for (int j = 0; j < 4; j++) qf[j] = __builtin_bit_cast(v8, *(const u32x4*)(Q + 8 * j));

    f32x4 o[8];
#pragma unroll
    for (int db = 0; db < 8; db++) o[db] = f32x4{0};
    float m = -__builtin_inff(), l = 0.f;
    const float C = a.scale_log2;
    for (int p = p0 + w; p < p1; p += 4) {
        int page = __builtin_amdgcn_readfirstlane(kv_page(a.b, it.b, p));
        const bool none = !kv_in_pool(a.b, page);
        if (none) {  // a page outside the pool: its keys are left out
            if (lane == 0 && kh == 0) atomicAdd(a.b.bad, 1ull);
            page = 0;
        }
        const uint8_t* blk = a.b.data + kv_block(a.b, page, kh);
        const uint32_t flag = a.b.flags[page];
        u32x4 kc[4], vc[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            kc[t] = *(const u32x4*)(blk + 1024 * t + 16 * lane);
            vc[t] = *(const u32x4*)(blk + LTX_KV_V + 1024 * t + 16 * lane);
        }
        const uint32_t ks = *(const uint32_t*)(blk + LTX_KV_KS + 4 * lane);
        u32x4 vs = *(const u32x4*)(blk + LTX_KV_VS + 64 * (r >> 2) + 16 * h);

        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float f = scale_of(ks, t);
            s[t] = f32x4{0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t x = kc[t][j];
                const u32x4 d = {Fp4<T>::template pair<0>(x, f), Fp4<T>::template pair<1>(x, f),
                                 Fp4<T>::template pair<2>(x, f), Fp4<T>::template pair<3>(x, f)};
                s[t] = Op<T>::mfma16(__builtin_bit_cast(v8, d), qf[j], s[t]);
            }
        }
        if (flag) kv_set_nan(s, kv_drop_nan(vs));
        if (none || (p + 1) * LTX_KV_PAGE > all) kv_mask(s, p, none ? 0 : mine, h);
        uint32_t pw[4][2];
        float corr;
        if (kv_softmax<T>(s, C, m, l, pw, corr))
#pragma unroll
            for (int db = 0; db < 8; db++) o[db] *= corr;
#pragma unroll
        for (int cc = 0; cc < 2; cc++) {
            const v8 pf = __builtin_bit_cast(v8, (u32x4){pw[2 * cc][0], pw[2 * cc][1], pw[2 * cc + 1][0],
                                                         pw[2 * cc + 1][1]});
            uint32_t x[8], f[2] = {vs[2 * cc], vs[2 * cc + 1]};
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = vc[2 * cc + (e >> 2)][e & 3];
            auto two = [&](auto B) {  // dims 8 r + 2 B and + 1: eight keys each
                constexpr int b = decltype(B)::value;
                u32x4 lo, hi;
                kv_v_pair<T, b>(x, f, lo, hi);
                o[2 * b] = Op<T>::mfma16(__builtin_bit_cast(v8, lo), pf, o[2 * b]);
                o[2 * b + 1] = Op<T>::mfma16(__builtin_bit_cast(v8, hi), pf, o[2 * b + 1]);
            };
            two(std::integral_constant<int, 0>{});
            two(std::integral_constant<int, 1>{});
            two(std::integral_constant<int, 2>{});
            two(std::integral_constant<int, 3>{});
        }
    }

    // the four waves' results into one: lane (r, h) holds dims 8 (4 h + i) + db
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
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
    const int col = tid >> 4, d0 = 8 * (tid & 15);
    if (col >= cols) return;
    float M = fmaxf(fmaxf(sm[0][col], sm[1][col]), fmaxf(sm[2][col], sm[3][col]));
    const float Mz = M == -__builtin_inff() ? 0.f : M;
    float lt = 0.f, x[8] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float f = __builtin_amdgcn_exp2f(sm[j][col] - Mz);
        lt = __builtin_fmaf(sl[j][col], f, lt);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(so[j][col][d0 + e], f, x[e]);
    }
    const int64_t cc = c0 + col;
    const int orow = (int)(cc / a.group), ohead = kh * a.group + (int)(cc % a.group);
    if (kv_runs(np, per) > 1) {
        const size_t at = ((size_t)blockIdx.x * a.b.kvh + kh) * KV_TILE + col;
        float* ml = a.part + 2 * at;
        float* po = a.part + 2 * (size_t)a.items * a.b.kvh * KV_TILE + at * LTX_HD + d0;
        if (d0 == 0) *(f32x2*)ml = f32x2{M, lt};
        *(f32x4*)po = f32x4{x[0], x[1], x[2], x[3]};
        *(f32x4*)(po + 4) = f32x4{x[4], x[5], x[6], x[7]};
        return;
    }
    const int grow = it.s.s0 + orow;
    const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)grow * a.heads + ohead]) : 1.0f;
    const float f = kv_limit(a.causal, it.s, orow) > 0 ? g / lt : 0.f;
    u32x4 out;
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = Op<T>::cvt2(x[2 * e] * f, x[2 * e + 1] * f);
    *(u32x4*)((uint16_t*)a.out + (size_t)grow * a.ldo + (size_t)ohead * LTX_HD + d0) = out;
}

extern "C" __global__ void __launch_bounds__(256) ltx_kv_attn_f16(const LtxKvAttnArgs a) { kv_attn<_Float16>(a); }
extern "C" __global__ void __launch_bounds__(256) ltx_kv_attn_bf16(const LtxKvAttnArgs a) { kv_attn<__bf16>(a); }

// Many columns: a workgroup takes 128 NQ columns, its eight waves 16 NQ each, and a
// run of pages. A page's codes become MFMA operands once for all eight waves, in LDS,
// in the order the operands are read (16 bytes a lane, no conflicts): waves 0 .. 3 a
// 16-key block of K each, waves 4 .. 7 half the dims of 32 keys of V each, one page
// ahead, from codes loaded two pages ahead. One barrier a page.
template <typename T, int NQ>
__device__ __forceinline__ void kv_attn_rows(const LtxKvAttnArgs& a) {
    typedef typename Op<T>::v8 v8;
    __shared__ __attribute__((aligned(1024))) uint8_t sk[2][16384];
    __shared__ __attribute__((aligned(1024))) uint8_t sv[2][16384];
    __shared__ uint32_t snan[2][2][4];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the items of a cached head follow each other on one XCD
    const int total = a.items * a.b.kvh, id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (id >= total) return;
    const int kh = id / a.items, item = id - kh * a.items;
    const int per = kv_per(a);
    KvItem it;
    if (!kv_item(a, per, item, it)) return;
    const int limit = kv_tile_limit(a.causal, it.s, a.group, it.tile, a.tile), np = kv_pages(limit);
    const int p0 = it.run * per, p1 = min(np, p0 + min(per, np));
    if (it.run > 0 && p0 >= np) return;

    const int64_t ncol = (int64_t)it.s.n * a.group;
    const int64_t c0 = (int64_t)it.tile * a.tile + 16 * NQ * w;  // the wave's first column
    const bool idle = c0 >= ncol;
    int row[NQ], head[NQ], mine[NQ];
    v8 qf[NQ][4];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int64_t c = min(c0 + 16 * q + r, ncol - 1);
        row[q] = (int)(c / a.group);
        head[q] = kh * a.group + (int)(c % a.group);
        mine[q] = kv_limit(a.causal, it.s, row[q]);
        const uint16_t* Q =
            (const uint16_t*)a.q + (size_t)(it.s.s0 + row[q]) * a.ldq + (size_t)head[q] * LTX_HD + 32 * h;
#pragma unroll
        for (int j = 0; j < 4; j++) qf[q][j] = __builtin_bit_cast(v8, *(const u32x4*)(Q + 8 * j));
    }
    const int all = kv_limit(a.causal, it.s, (int)(min(c0, ncol - 1) / a.group));  // keys that every column sees
    const int most = kv_limit(a.causal, it.s, (int)((min(c0 + 16 * NQ, ncol) - 1) / a.group));  // or any does

    // staging: a page's index and flag, 64 pages a lane each
    int ids = 0;
    uint32_t flags = 0;
    auto look_up = [&](int p) {
        const int at = p + lane;
        ids = at < p1 ? kv_page(a.b, it.b, at) : 0;
        const bool none = !kv_in_pool(a.b, ids);
        if (none) {
            if (w == 0 && kh == 0) atomicAdd(a.b.bad, 1ull);
            ids = 0;
        }
        flags = a.b.flags[ids] ? 1u : 0u;
        if (none) flags |= 2u;
    };
    u32x4 x0, x1;
    uint32_t y0, y1, fl[2];  // codes and scales in flight; the flags of their page, and of the page in LDS
    const int vt = 2 * ((w - 4) >> 1);  // V: first 16-key block of the wave's 32 keys
    auto load = [&](int p) {
        if (((p - p0) & 63) == 0) look_up(p);
        const int l = (p - p0) & 63;
        const int page = __builtin_amdgcn_readlane(ids, l);
        fl[0] = __builtin_amdgcn_readlane(flags, l);
        const uint8_t* blk = a.b.data + kv_block(a.b, page, kh);
        if (w < 4) {
            x0 = *(const u32x4*)(blk + 1024 * w + 16 * lane);
            y0 = *(const uint32_t*)(blk + LTX_KV_KS + 4 * lane);
        } else {
            x0 = *(const u32x4*)(blk + LTX_KV_V + 1024 * vt + 16 * lane);
            x1 = *(const u32x4*)(blk + LTX_KV_V + 1024 * vt + 1024 + 16 * lane);
            const u32x2 y = *(const u32x2*)(blk + LTX_KV_VS + 64 * (r >> 2) + 16 * h + 4 * vt);
            y0 = y[0];
            y1 = y[1];
        }
    };
    auto stage = [&](int buf) {
        if (w < 4) {
            const float f = __builtin_bit_cast(float, ((y0 >> (8 * w)) & 255u) << 23);
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(u32x4*)(sk[buf] + 1024 * (4 * w + j) + 16 * lane) =
                    u32x4{Fp4<T>::template pair<0>(x0[j], f), Fp4<T>::template pair<1>(x0[j], f),
                          Fp4<T>::template pair<2>(x0[j], f), Fp4<T>::template pair<3>(x0[j], f)};
        } else {
            if (fl[0] & 1u) {
                u32x4 vs = {y0, y1, 0, 0};
                const uint32_t bits = kv_drop_nan(vs);
                y0 = vs[0];
                y1 = vs[1];
                if ((w & 1) == 0 && r == 0) snan[buf][vt >> 1][h] = bits;
            }
            const uint32_t x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]}, f[2] = {y0, y1};
            uint8_t* d = sv[buf] + 1024 * (4 * vt) + 16 * lane;
            u32x4 lo, hi;
            if ((w & 1) == 0) {
                kv_v_pair<T, 0>(x, f, lo, hi);
                *(u32x4*)d = lo;
                *(u32x4*)(d + 1024) = hi;
                kv_v_pair<T, 1>(x, f, lo, hi);
                *(u32x4*)(d + 2048) = lo;
                *(u32x4*)(d + 3072) = hi;
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

    f32x4 o[8][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
#pragma unroll
        for (int db = 0; db < 8; db++) o[db][q] = f32x4{0};
        m[q] = -__builtin_inff();
        l[q] = 0.f;
    }
    const float C = a.scale_log2;
    if (p0 < p1) {
        load(p0);
        stage(0);
        fl[1] = fl[0];
        if (p0 + 1 < p1) load(p0 + 1);
    }
    __syncthreads();
    for (int p = p0; p < p1; p++) {
        const int buf = (p - p0) & 1;
        const uint32_t flag = fl[1];
        const bool busy = !idle && p * LTX_KV_PAGE < most;
        f32x4 s[NQ][4];
        if (busy) {
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int t = 0; t < 4; t++) s[q][t] = f32x4{0};
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const v8 kf = __builtin_bit_cast(v8, *(const u32x4*)(sk[buf] + 1024 * (4 * t + j) + 16 * lane));
#pragma unroll
                    for (int q = 0; q < NQ; q++) s[q][t] = Op<T>::mfma16(kf, qf[q][j], s[q][t]);
                }
        }
        // the next page into the other buffer, the one after it on its way
        if (p + 1 < p1) {
            stage(buf ^ 1);
            fl[1] = fl[0];
            if (p + 2 < p1) load(p + 2);
        }
        if (busy) {
            if (flag & 1u) {
                const uint32_t bits = snan[buf][0][h] | snan[buf][1][h] << 8;
#pragma unroll
                for (int q = 0; q < NQ; q++) kv_set_nan(s[q], bits);
            }
            if ((flag & 2u) || (p + 1) * LTX_KV_PAGE > all)
#pragma unroll
                for (int q = 0; q < NQ; q++) kv_mask(s[q], p, flag & 2u ? 0 : mine[q], h);
            v8 pf[NQ][2];
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                uint32_t pw[4][2];
                float corr;
                if (kv_softmax<T>(s[q], C, m[q], l[q], pw, corr))
#pragma unroll
                    for (int db = 0; db < 8; db++) o[db][q] *= corr;
#pragma unroll
                for (int c = 0; c < 2; c++)
                    pf[q][c] = __builtin_bit_cast(v8, (u32x4){pw[2 * c][0], pw[2 * c][1], pw[2 * c + 1][0],
                                                              pw[2 * c + 1][1]});
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int db = 0; db < 8; db++) {
                    const v8 vf = __builtin_bit_cast(v8, *(const u32x4*)(sv[buf] + 1024 * (8 * c + db) + 16 * lane));
#pragma unroll
                    for (int q = 0; q < NQ; q++) o[db][q] = Op<T>::mfma16(vf, pf[q][c], o[db][q]);
                }
        }
        __syncthreads();
    }

    if (idle) return;
    const bool whole = kv_runs(np, per) == 1;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        if (c0 + 16 * q + r >= ncol) continue;
        float lt = l[q] + __shfl_xor(l[q], 16, 64);
        lt += __shfl_xor(lt, 32, 64);
        if (!whole) {
            const size_t at = ((size_t)item * a.b.kvh + kh) * a.tile + 16 * (NQ * w + q) + r;
            float* po = a.part + 2 * (size_t)a.items * a.b.kvh * a.tile + at * LTX_HD + 32 * h;
            if (h == 0) *(f32x2*)(a.part + 2 * at) = f32x2{m[q], lt};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                *(f32x4*)(po + 8 * i) = f32x4{o[0][q][i], o[1][q][i], o[2][q][i], o[3][q][i]};
                *(f32x4*)(po + 8 * i + 4) = f32x4{o[4][q][i], o[5][q][i], o[6][q][i], o[7][q][i]};
            }
            continue;
        }
        const int grow = it.s.s0 + row[q];
        const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)grow * a.heads + head[q]]) : 1.0f;
        const float f = mine[q] > 0 ? g / lt : 0.f;
        uint16_t* out = (uint16_t*)a.out + (size_t)grow * a.ldo + (size_t)head[q] * LTX_HD + 32 * h;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = Op<T>::cvt2(o[2 * e][q][i] * f, o[2 * e + 1][q][i] * f);
            *(u32x4*)(out + 8 * i) = v;
        }
    }
}

#define KV_ATTN_ROWS(NAME, T, NQ) \
    extern "C" __global__ void __launch_bounds__(512) NAME(const LtxKvAttnArgs a) { kv_attn_rows<T, NQ>(a); }
KV_ATTN_ROWS(ltx_kv_attn_f16_rows1, _Float16, 1)
KV_ATTN_ROWS(ltx_kv_attn_bf16_rows1, __bf16, 1)
KV_ATTN_ROWS(ltx_kv_attn_f16_rows2, _Float16, 2)
KV_ATTN_ROWS(ltx_kv_attn_bf16_rows2, __bf16, 2)

// The runs of a tile into one: a wave takes a row and query head.
template <typename T>
__device__ void kv_join(const LtxKvAttnArgs& a) {
    const int lane = threadIdx.x & 63, row = blockIdx.x, head = 4 * blockIdx.y + (threadIdx.x >> 6);
    if (head >= a.heads) return;
    const int b = __builtin_amdgcn_readfirstlane(kv_find(a.b, row, 0));
    if (b >= a.b.nseq) return;
    const KvSeq s = kv_seq(a.b, b);
    const int i = row - s.s0, kh = head / a.group;
    if (i < 0 || i >= s.n) return;
    const int per = kv_per(a);
    uint64_t base = 0;  // items of the sequences before
    if (b > 0) {
        for (int j = lane; j < b; j += 64) {
            const KvSeq q = kv_seq(a.b, j);
            base += (uint64_t)kv_tiles(q.n, a.group, a.tile) * kv_runs(kv_pages(q.L), per);
        }
        base = wave_sum(base);
    }
    const int64_t c = (int64_t)i * a.group + head % a.group;
    const int tile = (int)(c / a.tile), col = (int)(c % a.tile);
    const int runs = kv_runs(kv_pages(kv_tile_limit(a.causal, s, a.group, tile, a.tile)), per);
    const uint64_t item = base + (uint64_t)(kv_tiles(s.n, a.group, a.tile) - 1 - tile) * kv_runs(kv_pages(s.L), per);
    if (runs <= 1 || item + runs > (uint64_t)a.items) return;
    const float* ml = a.part + 2 * ((item * a.b.kvh + kh) * a.tile + col);
    const float* po = a.part + 2 * (size_t)a.items * a.b.kvh * a.tile +
                      ((item * a.b.kvh + kh) * a.tile + col) * LTX_HD + 2 * lane;
    const size_t step = (size_t)a.b.kvh * a.tile;
    float M = -__builtin_inff();
    for (int j = 0; j < runs; j++) M = fmaxf(M, ml[2 * step * j]);
    const float Mz = M == -__builtin_inff() ? 0.f : M;
    float lt = 0.f, x0 = 0.f, x1 = 0.f;
    for (int j = 0; j < runs; j++) {
        const f32x2 v = *(const f32x2*)(ml + 2 * step * j), y = *(const f32x2*)(po + LTX_HD * step * j);
        const float f = __builtin_amdgcn_exp2f(v[0] - Mz);
        lt = __builtin_fmaf(v[1], f, lt);
        x0 = __builtin_fmaf(y[0], f, x0);
        x1 = __builtin_fmaf(y[1], f, x1);
    }
    const float g = a.glog ? 2.0f * sigmoid_f(a.glog[(size_t)row * a.heads + head]) : 1.0f;
    const float f = kv_limit(a.causal, s, i) > 0 ? g / lt : 0.f;
    *(uint32_t*)((uint16_t*)a.out + (size_t)row * a.ldo + (size_t)head * LTX_HD + 2 * lane) =
        Op<T>::cvt2(x0 * f, x1 * f);
}

extern "C" __global__ void __launch_bounds__(256) ltx_kv_join_f16(const LtxKvAttnArgs a) { kv_join<_Float16>(a); }
extern "C" __global__ void __launch_bounds__(256) ltx_kv_join_bf16(const LtxKvAttnArgs a) { kv_join<__bf16>(a); }
