// Attention of up to 16 rows a column over 32 tokens: records of the resident form, and
// fp16 / bf16 rows, as operands of 16x16x32 products; exceptions written over the decoded
// values; softmax and P V of a column.  Shared by the kernels that read tiles so.
#pragma once

#include "lq_resident.h"

namespace lq {

// P is held in fp16 times 2^10: weights down to 2^-24 of the largest keep their 11 bits
constexpr float kPShift = 10.0f;

typedef float f2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pair_h(float a, float b) {   // one v_cvt_pk_f16_f32, to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{a, b}), h2_t));
}

// eight bf16 -> eight fp16: exact between 2^-14 and 65504, where the operands of the fp16 products lie
__device__ __forceinline__ uint4 bf_to_h(const uint4& w) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = pair_h(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xffff0000u));
    return make_uint4(y[0], y[1], y[2], y[3]);
}

template <bool BF16>
__device__ __forceinline__ uint4 load_row8(const uint16_t* p) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    return BF16 ? bf_to_h(w) : w;
}

// tokens outside the word weigh 0, and 0 times a NaN or an infinity is a NaN: their V is cleared
__device__ __forceinline__ void clear_v(uint32_t word, int k8, uint32_t vp[4][8]) {
    const uint32_t own = word >> (8 * k8);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t keep = ((own >> (2 * k)) & 1u ? 0x0000ffffu : 0u) | ((own >> (2 * k + 1)) & 1u ? 0xffff0000u : 0u);
#pragma unroll
        for (int i = 0; i < 8; i++) vp[k][i] &= keep;
    }
}

template <typename T>
__device__ __forceinline__ T at32(const void* base, uint32_t bytes) {
    return *reinterpret_cast<const T*>(static_cast<const char*>(base) + bytes);
}

// Exceptions (vectors outside the 5-bit range): a block's entries lie in record order
// from its base.  The first 32 of both blocks are loaded with the tile, one a lane (lanes
// 0..31 of the first block's, 32..63 of the second's), from the bases and counts of a tile
// further on: taken when the masks are known, their latency would stand in every tile that
// has one (with outlier channels all of them: 32768 tokens, 16 rows a head, 5.6 % of K's
// vectors, 9 us more).  A tile's cost is that of writing them over the decoded values
// (25.3 us without any, 27.3 with one vector in 1200, 30.9 with outlier channels).
struct Meta {
    uint32_t h0, h1, base, count;   // of the lane's half
};

// the record of the lane's entry as the block's header has it: of the first seven
__device__ __forceinline__ uint32_t head_rec(const Meta& m, uint32_t lane) {
    return (uint32_t)(((((uint64_t)m.h1 << 32) | m.h0) >> 8) >> (8 * (lane & 7))) & 255u;
}
// exceptions of the block that has more; wave-uniform
__device__ __forceinline__ uint32_t most_of(const Meta& m) {
    return max((uint32_t)__builtin_amdgcn_readlane((int)m.count, 0), (uint32_t)__builtin_amdgcn_readlane((int)m.count, 32));
}
__device__ __forceinline__ uint4 load_entry(const lq_resident& r, const Meta& m, uint32_t lane) {
    const uint32_t e = lane & 31;
    const int64_t at = (int64_t)m.base + e;
    return reinterpret_cast<const uint4*>(r.exc)[e < m.count && at < r.exc_cap ? at : 0];
}
// an entry's eight values 2c as fp16 pairs of c (halving is exact)
__device__ __forceinline__ void exc_pairs(const uint4& w, uint32_t p[4]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2_t h = {(_Float16)(int16_t)(x[i] & 0xffffu), (_Float16)(int16_t)(x[i] >> 16)};
        p[i] = __builtin_bit_cast(uint32_t, h * (h2_t){(_Float16)0.5f, (_Float16)0.5f});
    }
}

// A lane's eight records of 32 tokens, four from rec[0] on and four from rec[1] on (record
// numbers within their blocks; hi: whether of the second block).  As K: vector lane / 4
// of tokens 4 (lane % 4) .. + 3 of both blocks; as V: vector lane % 16 of the eight
// tokens 8 (lane / 16) .. + 7.  One form for both, so that a wave's records take the same
// registers whichever it decodes.
struct Lay {
    uint32_t rec[2], hi[2];
};
__device__ __forceinline__ Lay lay_of(bool isk, uint32_t lane) {
    if (isk) return {{4 * lane, 4 * lane}, {0u, 1u}};
    const uint32_t r = 16 * (lane & 15) + 8 * ((lane >> 4) & 1), h = lane >> 5;
    return {{r, r + 4}, {h, h}};
}
struct Raw {
    uint4 a[2];
    uint32_t b[2];
    uint2 s[2];
    uint2 mask[2];   // exceptions of the records' group
};

// pairs vp[k][i] = dimension 8 n + i of the lane's tokens 2 k, 2 k + 1, without the scales
__device__ __forceinline__ void decode_v(const Raw& d, uint32_t vp[4][8]) {
    const uint32_t aw[8] = {d.a[0].x, d.a[0].y, d.a[0].z, d.a[0].w, d.a[1].x, d.a[1].y, d.a[1].z, d.a[1].w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t w = d.b[k >> 1];
        rec_pairs_tok(aw[2 * k], w >> (16 * (k & 1)), aw[2 * k + 1], w >> (16 * (k & 1) + 8), vp[k]);
#pragma unroll
        for (int i = 0; i < 8; i++) vp[k][i] = unbias(vp[k][i]);
    }
}
__device__ __forceinline__ void scale_v(const Raw& d, uint32_t word, int lane, uint32_t vp[4][8]) {
    const uint32_t sw[4] = {d.s[0].x, d.s[0].y, d.s[1].x, d.s[1].y};
#pragma unroll
    for (int k = 0; k < 4; k++) mul_pairs<8>(vp[k], sw[k]);
    if (word != ~0u) clear_v(word, lane >> 4, vp);
}

// The record of number k among a block's exceptions (there are as many): the k-th set bit
// of its masks m, found by halving.
__device__ __forceinline__ uint32_t nth_record(const uint2 m[4], uint32_t k) {
    uint2 w = m[0];
    uint32_t at = 0u;
#pragma unroll
    for (uint32_t c = 0; c < 3; c++) {
        const uint32_t n = __builtin_popcount(w.x) + __builtin_popcount(w.y);
        if (at == 64 * c && k >= n) {
            k -= n;
            w = m[c + 1];
            at += 64u;
        }
    }
    const uint32_t n = __builtin_popcount(w.x);
    const bool up = k >= n;
    uint32_t x = up ? w.y : w.x;
    k -= up ? n : 0u;
    at += up ? 32u : 0u;
#pragma unroll
    for (uint32_t s = 16; s; s >>= 1) {
        const uint32_t b = __builtin_popcount(x & ((1u << s) - 1u));
        const bool over = k >= b;
        x = over ? x >> s : x;
        k -= over ? b : 0u;
        at += over ? s : 0u;
    }
    return at;
}
// Masks of block lane / 32 of a tile: group c's in lane l0 + step c of the first register
// for its first block, in lane l1 + step c of the second for its second
__device__ __forceinline__ void half_masks(const uint2& a, int l0, const uint2& b, int l1, int step, int lane, uint2 m[4]) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t x0 = (uint32_t)__builtin_amdgcn_readlane((int)a.x, l0 + step * c), y0 = (uint32_t)__builtin_amdgcn_readlane((int)a.y, l0 + step * c);
        const uint32_t x1 = (uint32_t)__builtin_amdgcn_readlane((int)b.x, l1 + step * c), y1 = (uint32_t)__builtin_amdgcn_readlane((int)b.y, l1 + step * c);
        m[c] = lane >> 5 ? make_uint2(x1, y1) : make_uint2(x0, y0);
    }
}

__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// put(rec, e): the lane's entry (pairs e) over record rec of block lane / 32, for all
// entries of a tile, a block's by rounds of 32; `ent` has the first.  Which record an entry
// is stands in the block's header where neither block has more than seven, as most tiles.
template <typename M, typename P>
__device__ __forceinline__ void each_entry(const lq_resident& r, const Meta& m, uint4 ent, uint32_t most, int lane, M masks, P put) {
    uint2 mk[4];
    if (most > 7) masks(mk);
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < most; r0 += 32) {
        const uint32_t k = r0 + (lane & 31);
        if (r0) ent = load_entry(r, {0u, 0u, m.base + r0, m.count > r0 ? m.count - r0 : 0u}, lane);
        const uint32_t rec = most > 7 ? nth_record(mk, k) & 255u : head_rec(m, lane);
        if (k < m.count) {
            // an entry that the list had no room for is zero (numbers of entries are below 2^31)
            const uint32_t keep = m.base + k < (uint32_t)min(r.exc_cap, (int64_t)INT_MAX) ? ~0u : 0u;
            uint32_t e[4];
            exc_pairs(make_uint4(ent.x & keep, ent.y & keep, ent.z & keep, ent.w & keep), e);
            put(rec, e);
        }
    }
}

// K for the operands of k_tree_few: a lane has tokens 8 g + 2 i, + 1 (lane % 16 = 4 g + i)
// of vectors 4 c + lane / 16
struct KFew {
    uint2 a[4];
    uint32_t b[4];
    uint32_t s;
    uint2 mask;      // lanes 0..7: exceptions of block lane / 4, record group lane % 4
};

// Exceptions of a wave's decoded pairs: these go through 8 KB of LDS of the wave's own,
// where the lanes that hold the entries write over them, all at once.  (Pulled into the
// registers of the records' lanes, one record group after the other, they cost as much as
// decoding the tile: 32768 tokens, 16 rows a head, 30.4 us a call against 27.1; 25.3
// without any exception.)
// Over the pairs of K's records 2 c + y:
__device__ __forceinline__ void patch_k(const lq_resident& r, const KFew& d, const Meta& m, const uint4& ent, uint32_t most,
                                        int lane, u32x4_t* area, uint32_t p[8][4]) {
#pragma unroll
    for (int j = 0; j < 8; j++) area[64 * j + lane] = u32x4_t{p[j][0], p[j][1], p[j][2], p[j][3]};
    wave_lds_sync();
    each_entry(r, m, ent, most, lane,
        [&](uint2 mk[4]) __attribute__((always_inline)) { half_masks(d.mask, 0, d.mask, 4, 1, lane, mk); },
        [&](uint32_t rec, const uint32_t e[4]) __attribute__((always_inline)) {
            area[64 * (2 * (rec >> 6) + (rec & 1)) + 16 * ((rec >> 4) & 3) + 8 * (lane >> 5) + ((rec & 15) >> 1)] =
                u32x4_t{e[0], e[1], e[2], e[3]};
        });
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const u32x4_t w = area[64 * j + lane];
#pragma unroll
        for (int i = 0; i < 4; i++) p[j][i] = w[i];
    }
    wave_lds_sync();
}
// over the pairs of decode_v:
__device__ __forceinline__ void patch_v(const lq_resident& r, const Raw& d, const Meta& m, const uint4& ent, uint32_t most,
                                        int lane, u32x4_t* area, uint32_t vp[4][8]) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        area[64 * j + lane] = u32x4_t{vp[j >> 1][4 * (j & 1)], vp[j >> 1][4 * (j & 1) + 1], vp[j >> 1][4 * (j & 1) + 2],
                                      vp[j >> 1][4 * (j & 1) + 3]};
    wave_lds_sync();
    each_entry(r, m, ent, most, lane,
        [&](uint2 mk[4]) __attribute__((always_inline)) { half_masks(d.mask[0], 0, d.mask[0], 32, 4, lane, mk); },
        [&](uint32_t rec, const uint32_t e[4]) __attribute__((always_inline)) {
            const uint32_t tok = 16 * (lane >> 5) + (rec & 15);   // of the tile's 32: pair (tok / 2) % 4 of lane vector + 16 (tok / 8)
            uint16_t* w = reinterpret_cast<uint16_t*>(area + 64 * (tok & 6) + 16 * (tok >> 3) + (rec >> 4)) + (tok & 1);
#pragma unroll
            for (int i = 0; i < 8; i++) w[(i & 4) * 128 + (i & 3) * 2] = (uint16_t)(i & 1 ? e[i >> 1] >> 16 : e[i >> 1]);
        });
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const u32x4_t w = area[64 * j + lane];
#pragma unroll
        for (int i = 0; i < 4; i++) vp[j >> 1][4 * (j & 1) + i] = w[i];
    }
    wave_lds_sync();
}

// V of the lane's eight tokens as decode_v gives it, tokens outside the word cleared
template <bool BF16>
__device__ __forceinline__ void rows_v(const uint16_t* p, int64_t st, int64_t t, int have, uint32_t word, int lane,
                                       uint32_t vp[4][8]) {
    const int n = lane & 15, k8 = lane >> 4;
    uint4 w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = *reinterpret_cast<const uint4*>(p + (t + min(8 * k8 + j, have - 1)) * st + 8 * n);
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (BF16) w[j] = bf_to_h(w[j]);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint4 w0 = w[2 * k], w1 = w[2 * k + 1];
        const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            vp[k][2 * i] = __builtin_amdgcn_perm(x1[i], x0[i], 0x05040100u);
            vp[k][2 * i + 1] = __builtin_amdgcn_perm(x1[i], x0[i], 0x07060302u);
        }
    }
    if (word != ~0u) clear_v(word, k8, vp);
}

// maximum over the lanes that hold a row: lane and lane ^ 32, and for 16-row columns
// lane ^ 16 (swaps of lane halves and of rows of 16, without LDS)
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quarters_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// A row's reference m need not be its maximum: it is raised (and l and o rescaled) once
// a score passes it by more than kLazy, so that P stays below 2^(kPShift + kLazy), in
// fp16's range.  With 32 rows a wave some row finds a new maximum in nearly every tile;
// passing the old one by 2^5 is rare after the first.
constexpr float kLazy = 5.0f;

// The weights of two scores as fp16, added to the sum as they are rounded (fp32).
__device__ __forceinline__ uint32_t weights(float s0, float s1, float c0, float off, float& l) {
    const uint32_t p = pair_h(__builtin_amdgcn_exp2f(__builtin_fmaf(s0, c0, off)), __builtin_amdgcn_exp2f(__builtin_fmaf(s1, c0, off)));
    l = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, p), h2_t{(_Float16)1.f, (_Float16)1.f}, l, false);
    return p;
}

// The softmax and P V of one column of 16 rows and 32 tokens: s[y][i] is the score of
// token 8 (lane / 16) + 2 i + y, word the tokens that the lane's row sees (every: all of
// them, for every lane).
struct FewState {
    float m, l;      // reference (base 2), the lane's part of the sum
    f4_t o[8];       // O^T: column lane % 16; o[mm][i]: dimension 8 (4 (lane / 16) + i) + mm
};
constexpr float kScale2 = 1.4426950408889634f / 11.313708498984761f;   // log2(e) / sqrt(128)

// Scores that the row does not see to -inf, and the row's reference raised where they pass
// it; returns what is added to a score times kScale2 for the logarithm of its weight.
__device__ __forceinline__ float few_reference(f4_t s[2], uint32_t word, bool every, int lane, FewState& st) {
    if (!every) {
        const uint32_t own = word >> (8 * (lane >> 4));
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[y][i] = (own >> (2 * i + y)) & 1u ? s[y][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[i >> 2][i & 3]);
    const float mn = quarters_max(mx) * kScale2;
    if (__any(mn > st.m + kLazy)) {
        const float up = mn > st.m + kLazy ? mn : st.m;   // as in products
        const float al = up == st.m ? 1.f : __builtin_amdgcn_exp2f(st.m - up);
        st.l *= al;
#pragma unroll
        for (int mm = 0; mm < 8; mm++)
#pragma unroll
            for (int i = 0; i < 4; i++) st.o[mm][i] *= al;
        st.m = up;
    }
    return (st.m == -INFINITY ? 0.f : -st.m) + kPShift;
}
__device__ __forceinline__ void few_products(const uint32_t p[4], const uint32_t vp[4][8], FewState& st) {
    const h8_t pb = as_h8(p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int mm = 0; mm < 8; mm++)
        st.o[mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(vp[0][mm], vp[1][mm], vp[2][mm], vp[3][mm]), pb, st.o[mm],
                                                          0, 0, 0);
}
__device__ __forceinline__ void few_attend(f4_t s[2], uint32_t word, bool every, const uint32_t vp[4][8], int lane,
                                           FewState& st) {
    const float off = few_reference(s, word, every, lane, st);
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = weights(s[0][i], s[1][i], kScale2, off, st.l);   // in the order of the tokens
    few_products(p, vp, st);
}

}  // namespace lq
