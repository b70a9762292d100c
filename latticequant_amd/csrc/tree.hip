// Attention of drafted tokens (the nodes of a tree, or a chain) over a resident
// prefix, the fp16 / bf16 tail and the drafts themselves, for gfx950.
//
// Row r = node * group + g of a kv head is node `node` of query head
// kvh * group + g.  A row sees the prefix and tail tokens of its sequence
// (from start on, the tail up to its length), its own node and the node's
// ancestors.  With z = q . k log2(e) / sqrt(128) the row's output is
//   o = sum_t 2^(z_t - m) v_t / sum_t 2^(z_t - m),   m = max_t z_t,
// taken in one pass: m, the sum l and o are rescaled when m grows.
//
// Two kernels, both of eight waves per (kv head, block of rows, split of the tokens):
//
// k_tree_few, up to 32 rows: a wave takes 32-token tiles of its own, decodes their
// records straight into MFMA operands and holds one or two columns of 16 rows.
//   S^T = K Q^T     8 MFMA 16x16x32 a column: lane column n is row n, so a row's scores
//                   lie in four lanes; K row 4 g + i of product x is token 8 g + 2 i + x
//   O^T += V^T P^T  8 MFMA: with that order a lane's scores are the eight tokens
//                   8 (lane / 16) .. + 7 of the B operand: P never leaves its lane.
//                   MFMA mm's row n is dimension 8 n + mm, the order in which a lane has
//                   the eight dimensions of a decoded vector
// k_tree_many, more rows: two or four waves (a team) hold 32 rows each and share their
// tokens: a tile is decoded once into LDS, K as rows, V with its dimensions as rows.
//   S^T = K Q^T     8 MFMA 32x32x16 per 32 tokens, K's row m is token
//                   16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4: a lane's scores are
//                   tokens 16 s + 8 (lane / 32) .. + 7, the B operand of step s
//   O^T += V^T P^T  8 MFMA; V's LDS row 16 i + n is dimension 8 n + i
// Decoding 32 tokens of K and V is about 430 VALU instructions, a column's softmax 60
// (16 rows) or 110 (32 rows) and its 16 MFMA 256 or 512 cycles: with few rows the
// decode bounds the loop and sharing it through LDS costs more than it saves.
#include <climits>
#include <cmath>

#include "lq_device.h"
#include "lq_resident.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

typedef float f16_t __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8;
constexpr int kMaxNodes = LQ_TREE_MAX_NODES;
constexpr int kVisWords = kMaxNodes / 32;
constexpr int kKRow = 2 * kHd + 16;            // bytes of a token's K row in LDS: 68 words, so 16 lanes at 16 tokens touch all banks
constexpr int kVRow = 2 * 32 + 16;             // bytes of a dimension's V row (32 tokens): 20 words, likewise
constexpr int kSub = 32 * kKRow + kHd * kVRow; // bytes of 32 tokens
constexpr int kMRow = kHd + 4;                 // floats of a row in the merge of a workgroup's teams
constexpr int kRecF = 4 + kHd;                 // floats of a split record: m, l, 2 unused, o[128]
// P is held in fp16 times 2^10: weights down to 2^-24 of the largest keep their 11 bits
constexpr float kPShift = 10.0f;
constexpr float kEmpty = -1.0f;                // l of a row that sees nothing (padding node); a sum is never negative

struct Rows {
    const uint16_t* p;
    int64_t sb, sh, st;
};

struct TreeArgs {
    lq_resident k, v;
    int64_t t_prefix;
    Rows q, dk, dv, tk, tv;
    uint16_t* out;
    int64_t ob, oh, ot;
    const int32_t* parents;
    const int32_t* tail_len;
    const int32_t* start;
    int64_t tail_cap;
    int heads, group, nodes, rows, rb, nsp, tiles;   // rows = nodes * group; rb: row blocks; tiles: of 32 max(1, C / 2) tokens
    int np, nt;                                       // prefix and tail tiles (the draft's follow)
    float* rec;
};

// 32-bit mask of the tokens [lo, hi) of a tile's 32
__device__ __forceinline__ uint32_t range_word(int64_t lo, int64_t hi) {
    if (hi <= 0 || lo >= 32 || lo >= hi) return 0u;
    const uint32_t up = hi >= 32 ? ~0u : (1u << hi) - 1u;
    return lo <= 0 ? up : up & ~((1u << lo) - 1u);
}

// The 32 tokens of a subtile: where they are and which of them the sequence has.
struct Sub {
    int kind;        // 0 prefix, 1 tail, 2 draft
    int64_t t;       // first token within its kind
    uint32_t word;
};

template <int S>   // S subtiles per tile
__device__ __forceinline__ Sub sub_of(const TreeArgs& A, int tile, int u, int64_t len, int64_t start) {
    Sub s;
    if (tile < A.np) {
        s.kind = 0;
        s.t = ((int64_t)tile * S + u) * 32;
        s.word = range_word(start - s.t, A.t_prefix - s.t);
    } else if (tile < A.np + A.nt) {
        s.kind = 1;
        s.t = ((int64_t)(tile - A.np) * S + u) * 32;
        s.word = range_word(start - A.t_prefix - s.t, len - s.t);
    } else {
        s.kind = 2;
        s.t = ((int64_t)(tile - A.np - A.nt) * S + u) * 32;
        s.word = range_word(0, A.nodes - s.t);
    }
    return s;
}

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

// ------------------------------------------------------- 32 tokens to LDS --

__device__ __forceinline__ void put_k(char* lds, int tok, int vec, const uint4& w) {
    *reinterpret_cast<uint4*>(lds + tok * kKRow + vec * 16) = w;
}
// vector n of tokens 8 k8 .. 8 k8 + 7: pairs vp[k][i] = dimension 8 n + i of tokens 2 k, 2 k + 1
__device__ __forceinline__ void put_v(char* lds, int n, int k8, const uint32_t vp[4][8]) {
#pragma unroll
    for (int i = 0; i < 8; i++)
        *reinterpret_cast<uint4*>(lds + 32 * kKRow + (16 * i + n) * kVRow + 16 * k8) =
            make_uint4(vp[0][i], vp[1][i], vp[2][i], vp[3][i]);
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

// Records of 32 prefix tokens from t on, in flight.  The second block of the last tile
// may lie past the prefix: the last block is read in its place (its tokens are outside
// the tile's word).  A block's record of vector v and token s is number 16 v + s.
// Every address is a wave-uniform base and a lane's 32-bit offset.
struct Blocks {
    int64_t rb0;     // first block
    uint32_t d;      // 1, or 0 where the second block is clamped
};
__device__ __forceinline__ Blocks blocks_of(const lq_resident& r, int64_t hd, int64_t t, int64_t T) {
    return {hd * r.cap_blocks + t / kRB, t + kRB < T ? 1u : 0u};
}
template <typename T>
__device__ __forceinline__ T at32(const void* base, uint32_t bytes) {
    return *reinterpret_cast<const T*>(static_cast<const char*>(base) + bytes);
}

// Exceptions (vectors outside the 5-bit range): a block's entries lie in record order
// from its base, so an entry's number is the base plus the set bits of the block's
// masks before it.  Entries are loaded by all lanes at once (a lane without one reads
// the list's first) and selected: no lane waits for another's.
__device__ __forceinline__ uint4 exc_at(const lq_resident& r, bool mine, int64_t e) {
    return reinterpret_cast<const uint4*>(r.exc)[mine ? e : 0];
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
__device__ __forceinline__ void exc_select(bool any, bool mine, const uint4& w, uint32_t p[4]) {
    if (!any) return;   // wave-uniform
    uint32_t e[4];
    exc_pairs(w, e);
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = mine ? e[i] : p[i];
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
    uint32_t base;   // first exception entry of block lane % 2 (K), of the lane's block (V)
};
__device__ __forceinline__ void load_raw(const lq_resident& r, int64_t hd, int64_t t, int64_t T, const Lay& y, uint32_t bhi,
                                         Raw& d) {
    const Blocks B = blocks_of(r, hd, t, T);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t blk = y.hi[j] & B.d;
        d.a[j] = at32<uint4>(r.a + B.rb0 * 256, (blk * 256 + y.rec[j]) * 4);
        d.b[j] = at32<uint32_t>(r.b + B.rb0 * 256, blk * 256 + y.rec[j]);
        d.s[j] = at32<uint2>(r.scale + B.rb0 * kRB, (blk * kRB + (y.rec[j] & 15)) * 2);
        d.mask[j] = at32<uint2>(r.mask + B.rb0 * 4, (blk * 4 + (y.rec[j] >> 6)) * 8);
    }
    d.base = at32<uint32_t>(r.meta + B.rb0 * 4 + 2, (bhi & B.d) * 16);
}

__device__ __forceinline__ void stage_k(const lq_resident& r, const Raw& d, int lane, char* lds) {
    const int v = lane >> 2, t0 = 4 * (lane & 3);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint32_t aw[4] = {d.a[x].x, d.a[x].y, d.a[x].z, d.a[x].w};
        uint4 ex[4];
        uint32_t own = 0u;
        bool any[4] = {false, false, false, false};
        if (__any((d.mask[x].x | d.mask[x].y) != 0u)) {
            const uint64_t m = ((uint64_t)d.mask[x].y << 32) | d.mask[x].x;
            const int pc = __builtin_popcountll(m), at = 16 * (v & 3) + t0;
            uint32_t idx = (uint32_t)__builtin_amdgcn_readlane((int)d.base, x);
#pragma unroll
            for (int g = 0; g < 3; g++) idx += (lane >> 4) > g ? __builtin_amdgcn_readlane(pc, 16 * g) : 0;
            idx += __builtin_popcountll(m & ((1ull << at) - 1ull));
            own = (uint32_t)(m >> at) & 15u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t e = (int64_t)idx + __builtin_popcount(own & ((1u << i) - 1u));
                const bool mine = ((own >> i) & 1u) && e < r.exc_cap;
                if (!mine) own &= ~(1u << i);
                any[i] = __any(mine);
                if (any[i]) ex[i] = exc_at(r, mine, e);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t p[4];
            rec_pairs(aw[i], (d.b[x] >> (8 * i)) & 0xffu, p);
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = unbias(p[j]);
            exc_select(any[i], (own >> i) & 1u, ex[i], p);
            const uint32_t sw = i < 2 ? d.s[x].x : d.s[x].y;
            mul_pairs<4>(p, __builtin_amdgcn_perm(0u, sw, i & 1 ? 0x03020302u : 0x01000100u));
            put_k(lds, 16 * x + t0 + i, v, make_uint4(p[0], p[1], p[2], p[3]));
        }
    }
}

// pairs vp[k][i] = dimension 8 n + i of the lane's tokens 2 k, 2 k + 1
__device__ __forceinline__ void decode_v(const lq_resident& r, const Raw& d, uint32_t word, int lane, uint32_t vp[4][8]) {
    const uint32_t aw[8] = {d.a[0].x, d.a[0].y, d.a[0].z, d.a[0].w, d.a[1].x, d.a[1].y, d.a[1].z, d.a[1].w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t w = d.b[k >> 1];
        rec_pairs_tok(aw[2 * k], w >> (16 * (k & 1)), aw[2 * k + 1], w >> (16 * (k & 1) + 8), vp[k]);
#pragma unroll
        for (int i = 0; i < 8; i++) vp[k][i] = unbias(vp[k][i]);
    }
    if (__any((d.mask[0].x | d.mask[0].y) != 0u)) {
        const int n = lane & 15, k8 = lane >> 4, g = n >> 2;
        const uint64_t m = ((uint64_t)d.mask[0].y << 32) | d.mask[0].x;
        const int pc = __builtin_popcountll(m), s0 = 16 * (n & 3) + 8 * (k8 & 1);
        uint32_t idx = d.base;
#pragma unroll
        for (int c = 0; c < 3; c++) {
            const int lo = __builtin_amdgcn_readlane(pc, 4 * c), hi = __builtin_amdgcn_readlane(pc, 32 + 4 * c);
            idx += g > c ? ((k8 >> 1) ? hi : lo) : 0;
        }
        idx += __builtin_popcountll(m & ((1ull << s0) - 1ull));
        const uint32_t own = (uint32_t)(m >> s0) & 0xffu;
#pragma unroll 1
        for (int q0 = 0; q0 < 8; q0 += 2) {   // the lane's tokens q0, q0 + 1: pair row q0 / 2
            if (!__any((own >> q0) & 3u)) continue;
            const int64_t e = (int64_t)idx + __builtin_popcount(own & ((1u << q0) - 1u));
            const bool m0 = ((own >> q0) & 1u) && e < r.exc_cap;
            const int64_t e1 = e + ((own >> q0) & 1u);
            const bool m1 = ((own >> q0) & 2u) && e1 < r.exc_cap;
            const uint4 x0 = exc_at(r, m0, e), x1 = exc_at(r, m1, e1);
            uint32_t p0[4], p1[4];
            exc_pairs(x0, p0);
            exc_pairs(x1, p1);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (k != q0 >> 1) continue;   // wave-uniform
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t h0 = m0 ? (p0[i >> 1] >> (16 * (i & 1))) & 0xffffu : vp[k][i] & 0xffffu;
                    const uint32_t h1 = m1 ? (i & 1 ? p1[i >> 1] & 0xffff0000u : p1[i >> 1] << 16) : vp[k][i] & 0xffff0000u;
                    vp[k][i] = h0 | h1;
                }
            }
        }
    }
    const uint32_t sw[4] = {d.s[0].x, d.s[0].y, d.s[1].x, d.s[1].y};
#pragma unroll
    for (int k = 0; k < 4; k++) mul_pairs<8>(vp[k], sw[k]);
    if (word != ~0u) clear_v(word, lane >> 4, vp);
}

// K for the operands of k_tree_few: a lane has tokens 8 g + 2 i, + 1 (lane % 16 = 4 g + i)
// of vectors 4 c + lane / 16
struct KFew {
    uint2 a[4];
    uint32_t b[4];
    uint32_t s;
    uint2 mask;      // lanes 0..7: exceptions of block lane / 4, record group lane % 4
    uint32_t base;   // first exception entry of the lane's block
};
__device__ __forceinline__ void load_few(const lq_resident& r, int64_t hd, int64_t t, int64_t T, uint32_t lane, KFew& d) {
    const Blocks B = blocks_of(r, hd, t, T);
    const uint32_t row = lane & 15, kg = lane >> 4, blk = (row >> 3) & B.d;
    const uint32_t tok = 8 * ((row >> 2) & 1) + 2 * (row & 3);   // in its block
    const uint32_t rec = blk * 256 + 16 * kg + tok;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        d.a[c] = at32<uint2>(r.a + B.rb0 * 256, rec * 4 + 256 * c);
        d.b[c] = at32<uint16_t>(r.b + B.rb0 * 256, rec + 64 * c);
    }
    d.s = at32<uint32_t>(r.scale + B.rb0 * kRB, (blk * kRB + tok) * 2);
    d.base = at32<uint32_t>(r.meta + B.rb0 * 4 + 2, blk * 16);
    d.mask = at32<uint2>(r.mask + B.rb0 * 4, ((lane >> 2) & B.d) * 32 + (lane & 3) * 8);
}

// the exception entries of the lane's eight records: bit 2 c + y of own: token y of group c
struct ExcFew {
    uint4 e[4][2];
    uint32_t own, any;
};
__device__ __forceinline__ void exc_few(const lq_resident& r, const KFew& d, int lane, ExcFew& ex) {
    const int row = lane & 15, kg = lane >> 4;
    const int at = 16 * kg + 8 * ((row >> 2) & 1) + 2 * (row & 3);
    uint32_t idx = d.base;
    ex.own = ex.any = 0u;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t l0 = (uint32_t)__builtin_amdgcn_readlane((int)d.mask.x, c), h0 = (uint32_t)__builtin_amdgcn_readlane((int)d.mask.y, c);
        const uint32_t l1 = (uint32_t)__builtin_amdgcn_readlane((int)d.mask.x, 4 + c), h1 = (uint32_t)__builtin_amdgcn_readlane((int)d.mask.y, 4 + c);
        if ((l0 | h0 | l1 | h1) == 0u) continue;   // wave-uniform
        const uint64_t m = row >> 3 ? ((uint64_t)h1 << 32) | l1 : ((uint64_t)h0 << 32) | l0;
        const int64_t e = (int64_t)idx + __builtin_popcountll(m & ((1ull << at) - 1ull));
        const uint32_t two = (uint32_t)(m >> at) & 3u;
        const bool m0 = (two & 1u) && e < r.exc_cap, m1 = (two & 2u) && e + (two & 1u) < r.exc_cap;
        ex.e[c][0] = exc_at(r, m0, e);
        ex.e[c][1] = exc_at(r, m1, e + (two & 1u));
        ex.own |= ((m0 ? 1u : 0u) | (m1 ? 2u : 0u)) << (2 * c);
        ex.any |= (__any(m0) ? 1u : 0u) << (2 * c) | (__any(m1) ? 2u : 0u) << (2 * c);
        idx += row >> 3 ? __builtin_popcount(l1) + __builtin_popcount(h1) : __builtin_popcount(l0) + __builtin_popcount(h0);
    }
}

template <bool BF16>
__device__ void rows_k(const Rows& R, int64_t b, int64_t h, int64_t t, uint32_t word, int lane, char* lds) {
    const uint16_t* p = R.p + b * R.sb + h * R.sh;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int tok = 16 * x + (lane & 15);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int vec = 4 * c + (lane >> 4);
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if ((word >> tok) & 1u) w = load_row8<BF16>(p + (t + tok) * R.st + 8 * vec);
            put_k(lds, tok, vec, w);
        }
    }
}

// V of the lane's eight tokens as decode_v gives it; returns whether one of the wave's
// values is an infinity or a NaN
template <bool BF16>
__device__ __forceinline__ bool rows_v(const Rows& R, int64_t b, int64_t h, int64_t t, uint32_t word, int lane,
                                       uint32_t vp[4][8]) {
    const uint16_t* p = R.p + b * R.sb + h * R.sh;
    const int n = lane & 15, k8 = lane >> 4;
    uint32_t bad = 0u;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int tok = 8 * k8 + 2 * k;
        uint4 w0 = make_uint4(0u, 0u, 0u, 0u), w1 = w0;
        if ((word >> tok) & 1u) w0 = load_row8<BF16>(p + (t + tok) * R.st + 8 * n);
        if ((word >> (tok + 1)) & 1u) w1 = load_row8<BF16>(p + (t + tok + 1) * R.st + 8 * n);
        const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            vp[k][2 * i] = __builtin_amdgcn_perm(x1[i], x0[i], 0x05040100u);
            vp[k][2 * i + 1] = __builtin_amdgcn_perm(x1[i], x0[i], 0x07060302u);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            bad |= (uint32_t)((vp[k][i] & 0x7c00u) == 0x7c00u) | (uint32_t)((vp[k][i] & 0x7c000000u) == 0x7c000000u);
    }
    return __any(bad != 0u);
}

// ---------------------------------------------------------- 32 x 32 of it --

struct RowState {
    float m, l;      // running maximum (base 2), the lane's part of the sum
    f16_t o[4];      // O^T: column lane % 32, row of MFMA dt: V row 32 dt + 8 (i / 4) + 4 (lane / 32) + i % 4
};

// token of score register i of a lane, without its half's 8 (lane / 32)
constexpr int tok_of(int i) { return 16 * (i >> 3) + 4 * ((i >> 2) & 1) + (i & 3); }

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

// One subtile for the wave's 32 rows: word has the visible tokens of the lane's
// row; every: all of them, for every lane; odd (with DRAFT): V is not finite.
template <bool DRAFT>
__device__ __forceinline__ void sub_attend(const char* lds, const h8_t q[8], uint32_t word, bool every, bool odd,
                                           int lane, RowState& st) {
    const float c0 = 1.4426950408889634f / 11.313708498984761f;   // log2(e) / sqrt(128)
    const int n = lane & 31, g = lane >> 5;
    const int tok = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
    f16_t s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 8; c++) {
        const h8_t ka = *reinterpret_cast<const h8_t*>(lds + tok * kKRow + 32 * c + 16 * g);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, q[c], s, 0, 0, 0);
    }
    const uint32_t own = word >> (8 * g);
    if (!every) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = (own >> tok_of(i)) & 1u ? s[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
    const float mn = fmaxf(st.m, halves_max(mx) * c0);
    if (__any(mn > st.m)) {
        // a row that has seen nothing has m = -inf, l = 0 and o = 0
        const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - mn);
        st.l *= al;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) st.o[d][i] *= al;
        st.m = mn;
    }
    const float off = (mn == -INFINITY ? 0.f : -mn) + kPShift;
    float p[16];
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c0, off));
        l += p[i];
    }
    st.l += l;
    const char* vl = lds + 32 * kKRow;
    if (!DRAFT || !odd) {
#pragma unroll
        for (int sx = 0; sx < 2; sx++) {
            const h8_t pb = as_h8(pair_h(p[8 * sx + 0], p[8 * sx + 1]), pair_h(p[8 * sx + 2], p[8 * sx + 3]),
                                  pair_h(p[8 * sx + 4], p[8 * sx + 5]), pair_h(p[8 * sx + 6], p[8 * sx + 7]));
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const h8_t va = *reinterpret_cast<const h8_t*>(vl + (32 * d + n) * kVRow + 16 * (2 * sx + g));
                st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pb, st.o[d], 0, 0, 0);
            }
        }
        return;
    }
    // A draft's V with infinities or NaN: they reach the rows that see it and no others,
    // so the products are taken token by token.
#pragma unroll 1
    for (int t = 0; t < 32; t++) {
        float pv = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) pv = 8 * g + tok_of(i) == t ? p[i] : pv;
        const float other = __shfl_xor(pv, 32, 64);
        pv = ((t >> 3) & 1) == g ? pv : other;
        if ((word >> t) & 1u) {
#pragma unroll
            for (int d = 0; d < 4; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int row = 32 * d + 8 * (i >> 2) + 4 * g + (i & 3);
                    const _Float16 v = *reinterpret_cast<const _Float16*>(vl + row * kVRow + 2 * t);
                    st.o[d][i] = __builtin_fmaf(pv, (float)v, st.o[d][i]);
                }
        }
    }
}

// ------------------------------------------------------------------ kernel --

// vis[i]: node i and its ancestors, or nothing where its chain of parents does not end
// in a root (-1).  Pointer doubling: after round k the words hold 2^k generations.
__device__ void tree_words(const int32_t* __restrict__ parents, int n, uint32_t (*vis)[kVisWords], int* up, int tid) {
    const bool mine = tid < n;
    if (mine) {
        const int p = parents[tid];
        up[tid] = p == -1 ? -1 : p >= 0 && p < tid ? p : -2;
#pragma unroll
        for (int w = 0; w < kVisWords; w++) vis[tid][w] = w == tid >> 5 ? 1u << (tid & 31) : 0u;
    }
    __syncthreads();
    for (int k = 1; k < n; k *= 2) {
        int a = -1;
        uint32_t w[kVisWords];
        if (mine) {
            a = up[tid];
            if (a >= 0) {
#pragma unroll
                for (int i = 0; i < kVisWords; i++) w[i] = vis[a][i];
            }
        }
        const int next = mine && a >= 0 ? up[a] : a;
        __syncthreads();
        if (mine && a >= 0) {
            up[tid] = next;
#pragma unroll
            for (int i = 0; i < kVisWords; i++) vis[tid][i] |= w[i];
        }
        __syncthreads();
    }
    if (mine && up[tid] != -1) {
#pragma unroll
        for (int w = 0; w < kVisWords; w++) vis[tid][w] = 0u;
    }
    __syncthreads();
}

__device__ __forceinline__ void out_pair(const TreeArgs& A, bool bf16, int64_t b, int64_t kvh, int r, int d, float x,
                                         float y) {
    const int node = r / A.group, g = r % A.group;
    uint16_t* p = A.out + b * A.ob + (kvh * A.group + g) * A.oh + (int64_t)node * A.ot + d;
    *reinterpret_cast<uint32_t*>(p) = bf16 ? (uint32_t)f2bf(x) | ((uint32_t)f2bf(y) << 16)
                                           : (uint32_t)f2h(x) | ((uint32_t)f2h(y) << 16);
}

// Split sp's share of the tiles: `per` of the cache's, the draft's all to the last.
struct Share {
    int first, end;
};
__device__ __forceinline__ Share share_of(const TreeArgs& A, int sp) {
    const int per = (A.tiles + A.nsp - 1) / A.nsp, cache = A.np + A.nt;
    return {min(sp * per, cache), sp == A.nsp - 1 ? A.tiles : min((sp + 1) * per, cache)};
}

// The teams' (m, l, O) of a workgroup's rows (in s_m, s_l and buf by wave and column,
// COLS columns a wave, C waves a team) joined, to the record of the split or to out.
template <int C, int COLS, bool BF16>
__device__ __forceinline__ void join_teams(const TreeArgs& A, int64_t hd, int sp, int row0, const float* buf,
                                           const float (*s_m)[32], const float (*s_l)[32],
                                           const uint32_t (*vis)[kVisWords], int tid) {
    constexpr int T = kWaves / C;
    const bool last = sp == A.nsp - 1;
    for (int idx = tid; idx < COLS * C * (kHd / 2); idx += kWaves * 64) {
        const int lr = idx / (kHd / 2), d = 2 * (idx % (kHd / 2));
        const int rr = row0 + lr;
        if (rr >= A.rows) break;               // idx grows with the row
        const int w0 = lr / COLS, c = lr % COLS;
        float M = -INFINITY;
#pragma unroll
        for (int t = 0; t < T; t++) M = fmaxf(M, s_m[t * C + w0][c]);
        float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const int w = t * C + w0;
            const float f = s_m[w][c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w][c] - M);
            const float2 o = *reinterpret_cast<const float2*>(buf + (w * COLS + c) * kMRow + d);
            L += s_l[w][c] * f;
            x += o.x * f;
            y += o.y * f;
        }
        const int nd = rr / A.group;
        const bool empty = last && !((vis[nd][nd >> 5] >> (nd & 31)) & 1u);
        if (A.nsp == 1) {
            const float inv = 1.f / L;
            out_pair(A, BF16, hd / A.heads, hd % A.heads, rr, d, empty ? 0.f : x * inv, empty ? 0.f : y * inv);
        } else {
            float* rec = A.rec + ((hd * A.nsp + sp) * A.rows + rr) * kRecF;
            *reinterpret_cast<float2*>(rec + 4 + d) = make_float2(x, y);
            if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(M, empty ? kEmpty : L);
        }
    }
}

struct Place {       // what a workgroup works on
    int64_t hd, b, kvh, len, start;
    int sp, row0;
    int first;       // prefix tile (of 32 tokens) that holds the first visible token
};
__device__ __forceinline__ Place place_of(const TreeArgs& A, int rows_wg) {
    Place p;
    int64_t bid = blockIdx.x;
    p.row0 = (int)(bid % A.rb) * rows_wg;
    bid /= A.rb;
    p.sp = (int)(bid % A.nsp);
    p.hd = bid / A.nsp;
    p.b = p.hd / A.heads;
    p.kvh = p.hd % A.heads;
    p.len = A.tail_cap ? (A.tail_len ? min((int64_t)max(A.tail_len[p.b], 0), A.tail_cap) : A.tail_cap) : 0;
    p.start = A.start ? A.start[p.b] : 0;
    p.first = (int)(min(max(p.start, (int64_t)0), A.t_prefix) / 32);
    return p;
}

// 8 values of query row r from dimension d on
template <bool BF16>
__device__ __forceinline__ h8_t load_q(const TreeArgs& A, const Place& P, int r, int node, int d) {
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (r < A.rows)
        w = load_row8<BF16>(A.q.p + P.b * A.q.sb + (P.kvh * A.group + r % A.group) * A.q.sh + (int64_t)node * A.q.st + d);
    return __builtin_bit_cast(h8_t, w);
}

template <int C, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void k_tree_many(TreeArgs A) {
    constexpr int S = C / 2;                   // subtiles of a tile: waves 0 .. S - 1 of a team decode their K, the others V
    constexpr int T = kWaves / C;              // teams
    constexpr int kStage = T * S * kSub, kMerge = kWaves * 32 * kMRow * 4;
    __shared__ __align__(16) char s_buf[kStage > kMerge ? kStage : kMerge];
    __shared__ uint32_t s_vis[kMaxNodes][kVisWords];
    __shared__ int s_up[kMaxNodes];
    __shared__ int s_bad[T][S];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int team = wave / C, ct = wave % C;
    const Place P = place_of(A, 32 * C);
    if (P.sp == A.nsp - 1) tree_words(A.parents + P.b * A.nodes, A.nodes, s_vis, s_up, tid);

    // the wave's rows: column lane % 32
    const int r = P.row0 + 32 * ct + (lane & 31);
    const int node = r < A.rows ? r / A.group : 0;
    h8_t q[8];
#pragma unroll
    for (int c = 0; c < 8; c++) q[c] = load_q<BF16>(A, P, r, node, 16 * c + 8 * (lane >> 5));
    RowState st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) st.o[d][i] = 0.f;

    const Share sh = share_of(A, P.sp);
    char* buf = s_buf + team * S * kSub;
    const bool isk = ct < S;                   // wave-uniform
    const int mine = ct % S;                   // the subtile whose K or V the wave decodes
    const bool rows_here = P.row0 + 32 * ct < A.rows;
    const int split = min(sh.end, A.np);       // prefix tiles, then rows: two loops, each with the registers it needs
    int t0 = max(sh.first, P.first / S);
    if (t0 < split) {
        // The wave's records of its next tile are in flight while it works on this one.  The
        // reload is unconditional (past the share it reads the team's last tile again), so
        // that it lands in place; nothing waits on it before the next decode.
        const lq_resident& res = isk ? A.k : A.v;
        const Lay lay = lay_of(isk, lane);
        Raw raw;
        auto fetch = [&](int tile) {
            const int64_t t = min(((int64_t)min(tile, split - 1) * S + mine) * 32, A.t_prefix - kRB);
            load_raw(res, P.hd, t, A.t_prefix, lay, isk ? lane & 1 : lane >> 5, raw);
        };
        fetch(t0 + team);
        for (; t0 < split; t0 += T) {
            const int tile = t0 + team;
            const Sub sb = sub_of<S>(A, tile, mine, P.len, P.start);
            char* lds = buf + mine * kSub;
            if (isk) {
                stage_k(A.k, raw, lane, lds);
            } else {
                uint32_t vp[4][8];
                decode_v(A.v, raw, sb.word, lane, vp);
                put_v(lds, lane & 15, lane >> 4, vp);
            }
            __builtin_amdgcn_sched_barrier(0);   // every use of the records before their reload
            fetch(tile + T);
            __syncthreads();
            if (tile < split && rows_here) {
#pragma unroll 1
                for (int u = 0; u < S; u++) {
                    const Sub su = sub_of<S>(A, tile, u, P.len, P.start);
                    if (su.word) sub_attend<false>(buf + u * kSub, q, su.word, su.word == ~0u, false, lane, st);
                }
            }
            __syncthreads();
        }
    }
    for (t0 = max(sh.first, A.np); t0 < sh.end; t0 += T) {
        const int tile = t0 + team;
        if (tile < sh.end) {
            const Sub sb = sub_of<S>(A, tile, mine, P.len, P.start);
            char* lds = buf + mine * kSub;
            if (sb.word) {
                if (isk) {
                    rows_k<BF16>(sb.kind == 1 ? A.tk : A.dk, P.b, P.kvh, sb.t, sb.word, lane, lds);
                } else {
                    uint32_t vp[4][8];
                    const bool bad = rows_v<BF16>(sb.kind == 1 ? A.tv : A.dv, P.b, P.kvh, sb.t, sb.word, lane, vp);
                    put_v(lds, lane & 15, lane >> 4, vp);
                    if (lane == 0) s_bad[team][mine] = bad;
                }
            }
        }
        __syncthreads();
        if (tile < sh.end && rows_here) {
#pragma unroll 1
            for (int u = 0; u < S; u++) {
                const Sub sb = sub_of<S>(A, tile, u, P.len, P.start);
                if (!sb.word) continue;
                const bool draft = sb.kind == 2;
                const uint32_t w = draft ? sb.word & s_vis[node][sb.t >> 5] : sb.word;
                sub_attend<true>(buf + u * kSub, q, w, !draft && w == ~0u,
                                 draft && __builtin_amdgcn_readfirstlane(s_bad[team][u]), lane, st);
            }
        }
        __syncthreads();
    }

    const float l = st.l + __shfl_xor(st.l, 32, 64);
    if (lane < 32) {
        s_m[wave][lane] = st.m;
        s_l[wave][lane] = l;
    }
    float* dst = reinterpret_cast<float*>(s_buf) + (wave * 32 + (lane & 31)) * kMRow;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {          // vector 8 j + 4 (lane / 32) + i: dimensions 8 n + 2 d + h
            float* x = dst + 8 * (8 * j + 4 * (lane >> 5) + i);
            *reinterpret_cast<f4_t*>(x) = f4_t{st.o[0][4 * j + i], st.o[0][8 + 4 * j + i], st.o[1][4 * j + i],
                                               st.o[1][8 + 4 * j + i]};
            *reinterpret_cast<f4_t*>(x + 4) = f4_t{st.o[2][4 * j + i], st.o[2][8 + 4 * j + i], st.o[3][4 * j + i],
                                                   st.o[3][8 + 4 * j + i]};
        }
    __syncthreads();
    join_teams<C, 32, BF16>(A, P.hd, P.sp, P.row0, reinterpret_cast<const float*>(s_buf), s_m, s_l, s_vis, tid);
}

// The softmax and P V of one column of 16 rows and 32 tokens: s[y][i] is the score of
// token 8 (lane / 16) + 2 i + y, word the tokens that the lane's row sees (every: all of
// them, for every lane), odd (with DRAFT) that V is not finite.
struct FewState {
    float m, l;      // running maximum (base 2), the lane's part of the sum
    f4_t o[8];       // O^T: column lane % 16; o[mm][i]: dimension 8 (4 (lane / 16) + i) + mm
};
template <bool DRAFT>
__device__ __forceinline__ void few_attend(f4_t s[2], uint32_t word, bool every, bool odd, const uint32_t vp[4][8],
                                           int lane, FewState& st) {
    const float c0 = 1.4426950408889634f / 11.313708498984761f;   // log2(e) / sqrt(128)
    const int col = lane & 15, g = lane >> 4;
    if (!every) {
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[y][i] = (word >> (8 * g + 2 * i + y)) & 1u ? s[y][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[i >> 2][i & 3]);
    const float mn = fmaxf(st.m, quarters_max(mx) * c0);
    if (__any(mn > st.m)) {
        // a row that has seen nothing has m = -inf, l = 0 and o = 0
        const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - mn);
        st.l *= al;
#pragma unroll
        for (int mm = 0; mm < 8; mm++)
#pragma unroll
            for (int i = 0; i < 4; i++) st.o[mm][i] *= al;
        st.m = mn;
    }
    const float off = (mn == -INFINITY ? 0.f : -mn) + kPShift;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {              // in the order of the tokens
        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i & 1][i >> 1], c0, off));
        st.l += p[i];
    }
    if (!DRAFT || !odd) {
        const h8_t pb = as_h8(pair_h(p[0], p[1]), pair_h(p[2], p[3]), pair_h(p[4], p[5]), pair_h(p[6], p[7]));
#pragma unroll
        for (int mm = 0; mm < 8; mm++)
            st.o[mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(vp[0][mm], vp[1][mm], vp[2][mm], vp[3][mm]), pb,
                                                              st.o[mm], 0, 0, 0);
        return;
    }
    // A draft's V with infinities or NaN: they reach the rows that see it and no others, so
    // the products are taken token by token.
#pragma unroll 1
    for (int t = 0; t < 32; t++) {
        float pv = p[0];
#pragma unroll
        for (int i = 1; i < 8; i++) pv = (t & 7) == i ? p[i] : pv;
        pv = __shfl(pv, col + 16 * (t >> 3), 64);
        const bool see = (word >> t) & 1u;
#pragma unroll
        for (int mm = 0; mm < 8; mm++) {
            uint32_t w = vp[0][mm];
#pragma unroll
            for (int k = 1; k < 4; k++) w = ((t >> 1) & 3) == k ? vp[k][mm] : w;
            w = t & 1 ? w >> 16 : w & 0xffffu;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = h2f((uint16_t)__shfl((int)w, 4 * g + i + 16 * (t >> 3), 64));
                if (see) st.o[mm][i] = __builtin_fmaf(pv, v, st.o[mm][i]);
            }
        }
    }
}

// Up to 16 Q rows of a kv head, Q columns of 16 a wave, tokens dealt to the waves.
template <int Q, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void k_tree_few(TreeArgs A) {
    constexpr int N = 16 * Q;                  // nodes at most: a node has a row at least
    __shared__ __align__(16) float s_buf[kWaves * 16 * Q * kMRow];
    __shared__ uint32_t s_vis[N][kVisWords];
    __shared__ int s_up[N];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const Place P = place_of(A, 16 * Q);
    if (P.sp == A.nsp - 1) tree_words(A.parents + P.b * A.nodes, A.nodes, s_vis, s_up, tid);

    const Share sh = share_of(A, P.sp);
    const int split = min(sh.end, A.np);       // prefix tiles, then rows: two loops, each with the registers it needs
    // The records of the wave's next tile are in flight during the products of this one.  The
    // reload is unconditional (past the share it reads the last tile again), so that it
    // lands in place; nothing waits on it before the next decode.
    const Lay lay = lay_of(false, lane);
    KFew kr;
    Raw vr;
    auto fetch = [&](int tile) {
        const int64_t t = (int64_t)min(tile, split - 1) * 32;
        load_few(A.k, P.hd, t, A.t_prefix, lane, kr);
        load_raw(A.v, P.hd, t, A.t_prefix, lay, lane >> 5, vr);
    };
    int tile = max(sh.first, P.first) + wave;
    const bool prefix = max(sh.first, P.first) < split;
    if (prefix) fetch(tile);
    h8_t q[Q][4];
    int node[Q];
    FewState st[Q];
#pragma unroll
    for (int x = 0; x < Q; x++) {
        const int r = 16 * x + col;
        node[x] = r < A.rows ? r / A.group : 0;
#pragma unroll
        for (int c = 0; c < 4; c++) q[x][c] = load_q<BF16>(A, P, r, node[x], 32 * c + 8 * g);
        st[x].m = -INFINITY;
        st[x].l = 0.f;
#pragma unroll
        for (int mm = 0; mm < 8; mm++) st[x].o[mm] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    for (; tile < split; tile += kWaves) {
        const Sub sb = sub_of<1>(A, tile, 0, P.len, P.start);
        f4_t s[Q][2];
        uint32_t vp[4][8];
#pragma unroll
        for (int x = 0; x < Q; x++) s[x][0] = s[x][1] = f4_t{0.f, 0.f, 0.f, 0.f};
        ExcFew ex;
        exc_few(A.k, kr, lane, ex);
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
                uint32_t p[4];
                rec_pairs(y ? kr.a[c].y : kr.a[c].x, (kr.b[c] >> (8 * y)) & 0xffu, p);
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = unbias(p[i]);
                exc_select((ex.any >> (2 * c + y)) & 1u, (ex.own >> (2 * c + y)) & 1u, ex.e[c][y], p);
                mul_pairs<4>(p, __builtin_amdgcn_perm(0u, kr.s, y ? 0x03020302u : 0x01000100u));
#pragma unroll
                for (int x = 0; x < Q; x++)
                    s[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(p[0], p[1], p[2], p[3]), q[x][c], s[x][y], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);   // one record group's operands live at a time
        }
        decode_v(A.v, vr, sb.word, lane, vp);
        __builtin_amdgcn_sched_barrier(0);       // every use of the records before their reload: it lands in place
        fetch(tile + kWaves);
#pragma unroll
        for (int x = 0; x < Q; x++) few_attend<false>(s[x], sb.word, sb.word == ~0u, false, vp, lane, st[x]);
    }
    if (!prefix) tile = max(sh.first, split) + wave;
    for (; tile < sh.end; tile += kWaves) {
        const Sub sb = sub_of<1>(A, tile, 0, P.len, P.start);
        if (!sb.word) continue;
        f4_t s[Q][2];
        uint32_t vp[4][8];
        const Rows& R = sb.kind == 1 ? A.tk : A.dk;
        const uint16_t* p = R.p + P.b * R.sb + P.kvh * R.sh;
#pragma unroll
        for (int x = 0; x < Q; x++) s[x][0] = s[x][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int tok = 8 * (col >> 2) + 2 * (col & 3) + y;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if ((sb.word >> tok) & 1u) w = load_row8<BF16>(p + (sb.t + tok) * R.st + 32 * c + 8 * g);
#pragma unroll
                for (int x = 0; x < Q; x++)
                    s[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w), q[x][c], s[x][y], 0, 0, 0);
            }
        }
        const bool bad = rows_v<BF16>(sb.kind == 1 ? A.tv : A.dv, P.b, P.kvh, sb.t, sb.word, lane, vp);
        const bool draft = sb.kind == 2;
#pragma unroll
        for (int x = 0; x < Q; x++) {
            const uint32_t w = draft ? sb.word & s_vis[node[x]][sb.t >> 5] : sb.word;
            few_attend<true>(s[x], w, !draft && w == ~0u, draft && bad, vp, lane, st[x]);
        }
    }
#pragma unroll
    for (int x = 0; x < Q; x++) {
        float l = st[x].l + __shfl_xor(st[x].l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (lane < 16) {
            s_m[wave][16 * x + lane] = st[x].m;
            s_l[wave][16 * x + lane] = l;
        }
        const f4_t* o = st[x].o;
        float* dst = s_buf + (wave * 16 * Q + 16 * x + col) * kMRow;
#pragma unroll
        for (int i = 0; i < 4; i++) {          // vector 4 g + i
            *reinterpret_cast<f4_t*>(dst + 8 * (4 * g + i)) = f4_t{o[0][i], o[1][i], o[2][i], o[3][i]};
            *reinterpret_cast<f4_t*>(dst + 8 * (4 * g + i) + 4) = f4_t{o[4][i], o[5][i], o[6][i], o[7][i]};
        }
    }
    __syncthreads();
    join_teams<1, 16 * Q, BF16>(A, P.hd, P.sp, 0, s_buf, s_m, s_l, s_vis, tid);
}

// one wave per row: the splits' records of it, in order
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs A, int64_t n, int bf16) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= n) return;
    const int64_t hd = row / A.rows;
    const int r = (int)(row % A.rows);
    const float* rec = A.rec + (hd * A.nsp * A.rows + r) * kRecF;
    const int64_t step = (int64_t)A.rows * kRecF;
    float M = -INFINITY;
    for (int p = lane; p < A.nsp; p += 64) M = fmaxf(M, rec[p * step]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll 8
    for (int p = 0; p < A.nsp; p++) {
        const float2 ml = *reinterpret_cast<const float2*>(rec + p * step);
        const float2 v = *reinterpret_cast<const float2*>(rec + p * step + 4 + 2 * lane);
        const float f = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - M);
        L = __builtin_fmaf(ml.y, f, L);
        x = __builtin_fmaf(v.x, f, x);
        y = __builtin_fmaf(v.y, f, y);
    }
    const bool empty = rec[(A.nsp - 1) * step + 1] == kEmpty;
    const float inv = 1.f / L;
    out_pair(A, bf16 != 0, hd / A.heads, hd % A.heads, r, 2 * lane, empty ? 0.f : x * inv, empty ? 0.f : y * inv);
}

// ------------------------------------------------------------------- plan --

struct Plan {
    int c, rb, np, nt, nd, nsp;
};

// Waves of a team: as many 32-row columns as there are rows, four at most (their
// O is 64 registers each).  Splits: of the counts that leave one, the one whose
// longest CU has the fewest tiles; among those the fewest splits (records are
// written and read once more).
bool plan(int64_t n_seq, int64_t heads, int64_t nodes, int64_t group, int64_t t_prefix, int64_t tail_cap, Plan* p) {
    if (n_seq < 1 || heads < 1 || nodes < 1 || nodes > kMaxNodes || group < 1 || group > 16 || t_prefix < 0 ||
        t_prefix % kRB || tail_cap < 0 || t_prefix > INT_MAX / 2 || tail_cap > INT_MAX / 4)
        return false;
    const int64_t rows = nodes * group;
    p->c = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;   // 1: k_tree_few
    const int64_t s = p->c > 1 ? p->c / 2 : 1, teams = kWaves / p->c, tt = 32 * s;
    p->rb = (int)((rows + 32 * p->c - 1) / (32 * p->c));
    p->np = (int)((t_prefix + tt - 1) / tt);
    p->nt = (int)((tail_cap + tt - 1) / tt);
    p->nd = (int)((nodes + tt - 1) / tt);
    const int64_t base = n_seq * heads * p->rb;
    if (base > INT_MAX / 256) return false;
    const int64_t tiles = p->np + p->nt + p->nd;
    int64_t best = -1;
    for (int64_t n = 1; n <= 256 && (n - 1) * teams < tiles; n++) {
        const int64_t per = (tiles + n - 1) / n;
        const int64_t cost = ((base * n + 255) / 256) * ((per + teams - 1) / teams + 2);
        if (best < 0 || cost < best) {
            best = cost;
            p->nsp = (int)n;
        }
    }
    return true;
}

bool tree_res_ok(const lq_resident* r) {
    return r && r->a && r->b && r->mask && r->meta && r->scale && r->n_heads > 0 && r->cap_blocks > 0 && r->exc_cap >= 0;
}

bool rows_ok(const lq_rows* r) {
    return r && r->p && ((uintptr_t)r->p & 15) == 0 && r->stride_b % 8 == 0 && r->stride_h % 8 == 0 && r->stride_t % 8 == 0;
}

Rows rows_of(const lq_rows* r) { return {static_cast<const uint16_t*>(r->p), r->stride_b, r->stride_h, r->stride_t}; }

template <bool BF16>
void tree_launch(const TreeArgs& A, int c, int64_t grid, hipStream_t s) {
    const dim3 g((unsigned)grid), wg(kWaves * 64);
    if (c == 4) hipLaunchKernelGGL((k_tree_many<4, BF16>), g, wg, 0, s, A);
    else if (c == 2) hipLaunchKernelGGL((k_tree_many<2, BF16>), g, wg, 0, s, A);
    else if (A.rows > 16) hipLaunchKernelGGL((k_tree_few<2, BF16>), g, wg, 0, s, A);
    else hipLaunchKernelGGL((k_tree_few<1, BF16>), g, wg, 0, s, A);
}

}  // namespace

extern "C" {

int64_t lq_tree_attn_workspace(int64_t n_seq, int64_t heads, int64_t n_nodes, int group, int64_t t_prefix,
                               int64_t tail_cap) {
    Plan p;
    if (!plan(n_seq, heads, n_nodes, group, t_prefix, tail_cap, &p)) return -1;
    return p.nsp > 1 ? n_seq * heads * p.nsp * n_nodes * group * kRecF * (int64_t)sizeof(float) : 16;
}

int lq_resident_tree_attention(const lq_resident *k, const lq_resident *v, int64_t t_prefix, const lq_rows *q,
                               const lq_rows *draft_k, const lq_rows *draft_v, const int32_t *d_parents,
                               int64_t n_seq, int64_t n_nodes, int group, const lq_rows *tail_k, const lq_rows *tail_v,
                               int64_t tail_cap, const int32_t *d_tail_len, const int32_t *d_start, int dtype,
                               void *d_work, const lq_rows *out, hipStream_t s) {
    if (!k || !v || k->n_heads < 1 || n_seq < 1 || k->n_heads != v->n_heads || k->n_heads % n_seq || !d_parents ||
        !d_work || !rows_ok(q) || !rows_ok(draft_k) || !rows_ok(draft_v) || !rows_ok(out) ||
        (dtype != LQ_F16 && dtype != LQ_BF16))
        return LQ_ERR_ARG;
    if (tail_cap > 0 && (!rows_ok(tail_k) || !rows_ok(tail_v))) return LQ_ERR_ARG;
    if (t_prefix > 0 && (!tree_res_ok(k) || !tree_res_ok(v) || t_prefix > k->cap_blocks * kRB ||
                         t_prefix > v->cap_blocks * kRB))
        return LQ_ERR_ARG;
    const int64_t heads = k->n_heads / n_seq;
    Plan p;
    if (!plan(n_seq, heads, n_nodes, group, t_prefix, tail_cap, &p) || heads > INT_MAX) return LQ_ERR_ARG;
    TreeArgs A{};
    if (t_prefix > 0) { A.k = *k; A.v = *v; }
    A.t_prefix = t_prefix;
    A.q = rows_of(q);
    A.dk = rows_of(draft_k);
    A.dv = rows_of(draft_v);
    if (tail_cap > 0) { A.tk = rows_of(tail_k); A.tv = rows_of(tail_v); }
    A.out = static_cast<uint16_t*>(out->p);
    A.ob = out->stride_b;
    A.oh = out->stride_h;
    A.ot = out->stride_t;
    A.parents = d_parents;
    A.tail_len = d_tail_len;
    A.start = d_start;
    A.tail_cap = tail_cap;
    A.heads = (int)heads;
    A.group = group;
    A.nodes = (int)n_nodes;
    A.rows = (int)n_nodes * group;
    A.rb = p.rb;
    A.nsp = p.nsp;
    A.np = p.np;
    A.nt = p.nt;
    A.tiles = p.np + p.nt + p.nd;
    A.rec = static_cast<float*>(d_work);
    const int64_t grid = k->n_heads * p.nsp * p.rb;
    if (dtype == LQ_BF16) tree_launch<true>(A, p.c, grid, s);
    else tree_launch<false>(A, p.c, grid, s);
    if (p.nsp > 1) {
        const int64_t n = k->n_heads * A.rows;
        hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s, A, n, dtype == LQ_BF16);
    }
    return launch_status();
}

}  // extern "C"
