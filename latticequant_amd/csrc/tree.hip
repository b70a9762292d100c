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
// k_tree_many, more rows: two, four or eight waves (a team) hold 32 rows each and share their
// tokens: a tile is decoded once into LDS, K as rows, V with its dimensions as rows.
//   S^T = K Q^T     8 MFMA 32x32x16 per 32 tokens, K's row m is token
//                   16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4: a lane's scores are
//                   tokens 16 s + 8 (lane / 32) .. + 7, the B operand of step s
//   O^T += V^T P^T  8 MFMA; V's LDS row 16 i + n is dimension 8 n + i
// Decoding 32 tokens of K and V is about 430 VALU instructions, a column's softmax 60
// (16 rows) or 110 (32 rows) and its 16 MFMA 256 or 512 cycles: with few rows the
// decode bounds the loop and sharing it through LDS costs more than it saves.
#include <algorithm>
#include <climits>
#include <cmath>

#include "lq_device.h"
#include "lq_few.h"

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
    int np, nt, per;                                  // prefix and tail tiles (the draft's follow); tiles of a split's share
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
    int have;        // tokens from t on that exist, 32 at most
    uint32_t word;   // those that the sequence sees
};

template <int S>   // S subtiles per tile
__device__ __forceinline__ Sub sub_of(const TreeArgs& A, int tile, int u, int64_t len, int64_t start) {
    Sub s;
    if (tile < A.np) {
        s.kind = 0;
        s.t = ((int64_t)tile * S + u) * 32;
        s.have = (int)min(A.t_prefix - s.t, (int64_t)32);
        s.word = range_word(start - s.t, A.t_prefix - s.t);
    } else if (tile < A.np + A.nt) {
        s.kind = 1;
        s.t = ((int64_t)(tile - A.np) * S + u) * 32;
        s.have = (int)min(len - s.t, (int64_t)32);
        s.word = range_word(start - A.t_prefix - s.t, len - s.t);
    } else {
        s.kind = 2;
        s.t = ((int64_t)(tile - A.np - A.nt) * S + u) * 32;
        s.have = (int)min(A.nodes - s.t, (int64_t)32);
        s.word = range_word(0, A.nodes - s.t);
    }
    return s;
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

__device__ __forceinline__ Meta load_meta(const lq_resident& r, int64_t hd, int64_t t, int64_t T, uint32_t lane) {
    const Blocks B = blocks_of(r, hd, t, T);
    const uint4 w = at32<uint4>(r.meta + B.rb0 * 4, ((lane >> 5) & B.d) * 16);
    return {w.x, w.y, w.z, w.w};
}

// The records and metas of a wave's tiles in a loop over whole ones: bases that advance by
// a round at a time and offsets that stay, so a reload is its loads and little else.
struct Walk {
    const char *a, *b, *s, *m, *t;
    uint32_t left;   // rounds that are still to come
};
__device__ __forceinline__ Walk walk_of(const lq_resident& r, int64_t block, uint32_t rounds) {
    return {reinterpret_cast<const char*>(r.a + block * 256), reinterpret_cast<const char*>(r.b + block * 256),
            reinterpret_cast<const char*>(r.scale + block * kRB), reinterpret_cast<const char*>(r.mask + block * 4),
            reinterpret_cast<const char*>(r.meta + block * 4), rounds};
}
__device__ __forceinline__ void step(Walk& w, uint32_t blocks) {   // stays at the last round
    const uint32_t n = w.left ? blocks : 0u;
    w.left -= w.left ? 1u : 0u;
    w.a += n * 1024;
    w.b += n * 256;
    w.s += n * 32;
    w.m += n * 32;
    w.t += n * 16;
}
__device__ __forceinline__ void load_walk(const Walk& w, const Lay& y, Raw& d) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t blk = y.hi[j];
        d.a[j] = at32<uint4>(w.a, (blk * 256 + y.rec[j]) * 4);
        d.b[j] = at32<uint32_t>(w.b, blk * 256 + y.rec[j]);
        d.s[j] = at32<uint2>(w.s, (blk * kRB + (y.rec[j] & 15)) * 2);
        d.mask[j] = at32<uint2>(w.m, (blk * 4 + (y.rec[j] >> 6)) * 8);
    }
}
__device__ __forceinline__ Meta load_meta(const Walk& w, uint32_t lane) {
    const uint4 x = at32<uint4>(w.t, (lane >> 5) * 16);
    return {x.x, x.y, x.z, x.w};
}
__device__ __forceinline__ void load_raw(const lq_resident& r, int64_t hd, int64_t t, int64_t T, const Lay& y, Raw& d) {
    const Blocks B = blocks_of(r, hd, t, T);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t blk = y.hi[j] & B.d;
        d.a[j] = at32<uint4>(r.a + B.rb0 * 256, (blk * 256 + y.rec[j]) * 4);
        d.b[j] = at32<uint32_t>(r.b + B.rb0 * 256, blk * 256 + y.rec[j]);
        d.s[j] = at32<uint2>(r.scale + B.rb0 * kRB, (blk * kRB + (y.rec[j] & 15)) * 2);
        d.mask[j] = at32<uint2>(r.mask + B.rb0 * 4, (blk * 4 + (y.rec[j] >> 6)) * 8);
    }
}

__device__ __forceinline__ void stage_k(const Raw& d, int lane, char* lds) {
    const int v = lane >> 2, t0 = 4 * (lane & 3);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const uint32_t aw[4] = {d.a[x].x, d.a[x].y, d.a[x].z, d.a[x].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t p[4];
            rec_pairs(aw[i], (d.b[x] >> (8 * i)) & 0xffu, p);
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = unbias(p[j]);
            const uint32_t sw = i < 2 ? d.s[x].x : d.s[x].y;
            mul_pairs<4>(p, __builtin_amdgcn_perm(0u, sw, i & 1 ? 0x03020302u : 0x01000100u));
            put_k(lds, 16 * x + t0 + i, v, make_uint4(p[0], p[1], p[2], p[3]));
        }
    }
}

// The exceptions of 32 tokens whose records are staged in LDS, over the staged ones; the
// tokens' scales go through `scales`, 32 of the wave's own.
__device__ __forceinline__ void patch_lds(bool isk, const lq_resident& r, const Raw& d, const Meta& m, const uint4& ent,
                                          uint32_t word, int lane, uint2* scales, char* lds) {
    const uint32_t most = most_of(m);
    if (!most) return;
    wave_lds_sync();
    if (isk ? lane < 4 : (lane & 15) == 0) {   // four tokens each
#pragma unroll
        for (int j = 0; j < 2; j++) scales[isk ? lane + 4 * j : 2 * (lane >> 4) + j] = d.s[j];
    }
    wave_lds_sync();
    each_entry(r, m, ent, most, lane,
        [&](uint2 mk[4]) __attribute__((always_inline)) {
            half_masks(d.mask[0], 0, isk ? d.mask[1] : d.mask[0], isk ? 0 : 32, isk ? 16 : 4, lane, mk);
        },
        [&](uint32_t rec, uint32_t p[4]) __attribute__((always_inline)) {
            const uint32_t tok = 16 * (lane >> 5) + (rec & 15), v = rec >> 4;
            mul_pairs<4>(p, __builtin_amdgcn_perm(0u, reinterpret_cast<const uint16_t*>(scales)[tok], 0x01000100u));
            if (isk) {
                put_k(lds, tok, v, make_uint4(p[0], p[1], p[2], p[3]));
            } else if ((word >> tok) & 1u) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    *reinterpret_cast<uint16_t*>(lds + 32 * kKRow + (16 * i + v) * kVRow + 2 * tok) =
                        (uint16_t)(i & 1 ? p[i >> 1] >> 16 : p[i >> 1]);
            }
        });
}

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
    d.mask = at32<uint2>(r.mask + B.rb0 * 4, ((lane >> 2) & B.d) * 32 + (lane & 3) * 8);
}

// fp16 / bf16 rows: 32 tokens from t on, of which the first `have` exist (one at least);
// the others read the last that does.
template <bool BF16>
__device__ __forceinline__ void rows_k(const uint16_t* p, int64_t st, int64_t t, int have, int lane, char* lds) {
    uint4 w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int tok = 16 * (j >> 2) + (lane & 15);
        w[j] = *reinterpret_cast<const uint4*>(p + (t + min(tok, have - 1)) * st + 8 * (4 * (j & 3) + (lane >> 4)));
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        put_k(lds, 16 * (j >> 2) + (lane & 15), 4 * (j & 3) + (lane >> 4), BF16 ? bf_to_h(w[j]) : w[j]);
}

// A draft's infinities and NaN must reach the rows that see it and no others, but 0 times
// one of them is a NaN: they are cleared here, and join_teams adds them to the rows that
// see them.  Returns whether the wave has any.
__device__ __forceinline__ bool clear_odd(uint32_t vp[4][8]) {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool lo = (vp[k][i] & 0x7c00u) == 0x7c00u, hi = (vp[k][i] & 0x7c000000u) == 0x7c000000u;
            bad = bad || lo || hi;
            vp[k][i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
        }
    return __any(bad);
}

// ---------------------------------------------------------- 32 x 32 of it --

struct RowState {
    float m, l;      // reference (base 2), the lane's part of the sum
    f16_t o[4];      // O^T: column lane % 32, row of MFMA dt: V row 32 dt + 8 (i / 4) + 4 (lane / 32) + i % 4
};

// token of score register i of a lane, without its half's 8 (lane / 32)
constexpr int tok_of(int i) { return 16 * (i >> 3) + 4 * ((i >> 2) & 1) + (i & 3); }

// Scores of U subtiles for the wave's 32 rows: eight steps of U MFMA each, K read two
// steps ahead (left to itself the compiler reads each step's K just before it).
template <int U>
__device__ __forceinline__ void scores(const char* lds, const h8_t q[8], int lane, f16_t s[U]) {
    const int n = lane & 31, g = lane >> 5;
    const int tok = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
    const char* kl = lds + tok * kKRow + 16 * g;
    h8_t ka[3][U];
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int u = 0; u < U; u++) ka[c][u] = *reinterpret_cast<const h8_t*>(kl + u * kSub + 32 * c);
#pragma unroll
    for (int u = 0; u < U; u++) s[u] = f16_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 8; c++) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c < 6) ka[(c + 2) % 3][u] = *reinterpret_cast<const h8_t*>(kl + u * kSub + 32 * (c + 2));
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[c % 3][u], q[c], s[u], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Softmax and P V of U subtiles' scores.  The weights of a half subtile (16 tokens) are
// taken beside the products of the half before, V is read three products ahead.
template <int U>
__device__ __forceinline__ void products(const char* lds, const f16_t s[U], int lane, RowState& st) {
    const float c0 = 1.4426950408889634f / 11.313708498984761f;   // log2(e) / sqrt(128)
    const int n = lane & 31, g = lane >> 5;
    constexpr int N = 8 * U;                   // products: half h, 32 dimensions d: number 4 h + d
    const char* vl = lds + 32 * kKRow + n * kVRow + 16 * g;
    auto read = [&](int f) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8_t*>(vl + (f >> 3) * kSub + 32 * (f & 3) * kVRow + 32 * ((f >> 2) & 1));
    };
    h8_t va[4];
#pragma unroll
    for (int f = 0; f < 3; f++) va[f] = read(f);
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[u][i]);
    const float mn = halves_max(mx) * c0;
    if (__any(mn > st.m + kLazy)) {
        // only the rows that passed it: a row's roundings do not depend on the others of its
        // wave.  (One that has seen nothing has m = -inf, l = 0 and o = 0.)
        const float up = mn > st.m + kLazy ? mn : st.m;
        const float al = up == st.m ? 1.f : __builtin_amdgcn_exp2f(st.m - up);
        st.l *= al;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) st.o[d][i] *= al;
        st.m = up;
    }
    const float off = (st.m == -INFINITY ? 0.f : -st.m) + kPShift;
    uint32_t p[2][4];
#pragma unroll
    for (int i = 0; i < 4; i++) p[0][i] = weights(s[0][2 * i], s[0][2 * i + 1], c0, off, st.l);
#pragma unroll
    for (int f = 0; f < N; f++) {
        const int h = f >> 2, d = f & 3;
        if (f + 3 < N) va[(f + 3) & 3] = read(f + 3);
        st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[f & 3], as_h8(p[h & 1][0], p[h & 1][1], p[h & 1][2], p[h & 1][3]),
                                                         st.o[d], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (h + 1 < 2 * U) {
            const int u = (h + 1) >> 1, i = 8 * ((h + 1) & 1) + 2 * d;
            p[(h + 1) & 1][d] = weights(s[u][i], s[u][i + 1], c0, off, st.l);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

template <int U>
__device__ __forceinline__ void sub_attend(const char* lds, const h8_t q[8], int lane, RowState& st) {
    f16_t s[U];
    scores<U>(lds, q, lane, s);
    products<U>(lds, s, lane, st);
}

// one subtile of which the lane's row sees the tokens of word
__device__ __forceinline__ void sub_masked(const char* lds, const h8_t q[8], uint32_t word, int lane, RowState& st) {
    f16_t s[1];
    scores<1>(lds, q, lane, s);
    const uint32_t own = word >> (8 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < 16; i++) s[0][i] = (own >> tok_of(i)) & 1u ? s[0][i] : -INFINITY;
    products<1>(lds, s, lane, st);
}

// ------------------------------------------------------------------ kernel --

// vis[i]: node i and its ancestors, or nothing where its chain of parents does not end
// in a root (-1).  p: node tid's parent.  Pointer doubling: after round k the words hold
// 2^k generations.
__device__ void tree_words(int p, int n, uint32_t (*vis)[kVisWords], int* up, int tid) {
    const bool mine = tid < n;
    if (mine) {
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

// eight values of a row from dimension d on; none of a row that sees nothing
__device__ __forceinline__ void out8(const TreeArgs& A, bool bf16, int64_t b, int64_t kvh, int r, int d, const f4_t& x,
                                     const f4_t& y, bool empty) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (!empty) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = i < 2 ? x[2 * i] : y[2 * i - 4], v = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
            w[i] = bf16 ? (uint32_t)f2bf(u) | ((uint32_t)f2bf(v) << 16) : pair_h(u, v);
        }
    }
    const int node = r / A.group, g = r % A.group;
    *reinterpret_cast<uint4*>(A.out + b * A.ob + (kvh * A.group + g) * A.oh + (int64_t)node * A.ot + d) =
        make_uint4(w[0], w[1], w[2], w[3]);
}

// Split sp's share of the tiles: `per` of the cache's, the draft's besides to the last.
struct Share {
    int first, end;
};
__device__ __forceinline__ Share share_of(const TreeArgs& A, int sp) {
    const int cache = A.np + A.nt;
    return {min(sp * A.per, cache), sp == A.nsp - 1 ? A.tiles : min((sp + 1) * A.per, cache)};
}

struct Place {       // what a workgroup works on
    int64_t hd, b, kvh, len, start;
    int sp, row0;
    int first;       // prefix tile (of 32 tokens) that holds the first visible token
};
__device__ __forceinline__ Place place_of(const TreeArgs& A, int rows_wg) {
    Place p;
    const uint32_t rest = blockIdx.x / (uint32_t)A.rb, hd = rest / (uint32_t)A.nsp;
    p.row0 = (int)(blockIdx.x % (uint32_t)A.rb) * rows_wg;
    p.sp = (int)(rest % (uint32_t)A.nsp);
    p.hd = hd;
    p.b = hd / (uint32_t)A.heads;
    p.kvh = hd % (uint32_t)A.heads;
    p.len = A.tail_cap ? (A.tail_len ? min((int64_t)max(A.tail_len[p.b], 0), A.tail_cap) : A.tail_cap) : 0;
    p.start = A.start ? A.start[p.b] : 0;
    p.first = (int)(min(max(p.start, (int64_t)0), A.t_prefix) / 32);
    return p;
}

// The teams' (m, l, O) of a workgroup's rows (in s_m, s_l and buf by wave and column,
// COLS columns a wave, C waves a team) joined, to the record of the split or to out.
template <int C, int COLS, bool BF16>
__device__ __forceinline__ void join_teams(const TreeArgs& A, const Place& P, const float* buf, const float (*s_m)[32],
                                           const float (*s_l)[32],
                                           const uint32_t (*vis)[kVisWords], const int* odd, int tid) {
    constexpr int T = kWaves / C;
    const bool last = P.sp == A.nsp - 1;
    const int d = 8 * (tid & 15);              // 16 lanes a row, eight dimensions a lane
    for (int lr = tid >> 4; lr < COLS * C; lr += kWaves * 4) {
        const int rr = P.row0 + lr;
        if (rr >= A.rows) break;
        const int w0 = lr / COLS, c = lr % COLS;
        float m[T], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int t = 0; t < T; t++) {
            m[t] = s_m[t * C + w0][c];
            M = fmaxf(M, m[t]);
        }
        f4_t x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float f = m[t] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[t] - M);
            const float* o = buf + ((t * C + w0) * COLS + c) * kMRow + d;
            L += s_l[t * C + w0][c] * f;
            x += *reinterpret_cast<const f4_t*>(o) * f;
            y += *reinterpret_cast<const f4_t*>(o + 4) * f;
        }
        bool empty = false;
        if (last) {
            const int nd = rr / A.group;
            empty = !((vis[nd][nd >> 5] >> (nd & 31)) & 1u);
            if (*odd) {
                const uint16_t* p = A.dv.p + P.b * A.dv.sb + P.kvh * A.dv.sh + d;
                for (int t = 0; t <= nd; t++) {
                    if (!((vis[nd][t >> 5] >> (t & 31)) & 1u)) continue;
                    const uint4 w = load_row8<BF16>(p + t * A.dv.st);
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float v = h2f((uint16_t)(u[i >> 1] >> (16 * (i & 1))));
                        if (!(fabsf(v) < INFINITY)) (i < 4 ? x : y)[i & 3] += v;
                    }
                }
            }
        }
        if (A.nsp == 1) {
            const float inv = 1.f / L;
            out8(A, BF16, P.b, P.kvh, rr, d, x * inv, y * inv, empty);
        } else {
            float* rec = A.rec + ((P.hd * A.nsp + P.sp) * A.rows + rr) * kRecF;
            *reinterpret_cast<f4_t*>(rec + 4 + d) = x;
            *reinterpret_cast<f4_t*>(rec + 8 + d) = y;
            if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(M, empty ? kEmpty : L);
        }
    }
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
    constexpr int U = S < 2 ? S : 2;           // subtiles taken together
    constexpr int T = kWaves / C;              // teams
    constexpr int kStage = 2 * T * S * kSub;   // two tiles a team: one is read while the next is decoded
    static_assert(kStage >= kWaves * 32 * (kMRow + 2) * 4 && kStage >= kMaxNodes * 4, "the join and the tree fit the stage");
    __shared__ __align__(16) char s_buf[kStage];
    __shared__ uint32_t s_vis[kMaxNodes][kVisWords];
    __shared__ uint2 s_scale[kWaves][8];
    __shared__ int s_odd;                      // a draft's V has infinities or NaN
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int team = wave / C, ct = wave % C;
    const Place P = place_of(A, 32 * C);
    const Share sh = share_of(A, P.sp);
    char* buf = s_buf + team * 2 * S * kSub;
    const bool isk = ct < S;                   // wave-uniform
    const int mine = ct % S;                   // the subtile whose K or V the wave decodes
    const bool rows_here = P.row0 + 32 * ct < A.rows;
    // the share's tiles of the prefix that the sequence sees whole; the others (cut by its
    // start or by the prefix's end, the tail's, the draft's) follow in a loop of their own
    const int seen = max(sh.first, P.first / S);
    const int h1 = min(sh.end, (int)(A.t_prefix / (32 * S)));
    const int h0 = min(max(sh.first, (int)((max(P.start, (int64_t)0) + 32 * S - 1) / (32 * S))), max(h1, seen));
    const bool prefix = h0 < h1;

    // The wave's records of its next tile are in flight while it works on this one, and the
    // bases of the tile after.  Reloads are unconditional (past the share they read the
    // last tile again), so that they land in place and nothing waits on them before their use.
    const lq_resident& res = isk ? A.k : A.v;
    const Lay lay = lay_of(isk, lane);
    Raw raw;
    Meta meta, ahead;
    uint4 ent;
    // the team's rounds; a team without a tile in the last one reads that of the one before
    const uint32_t tiles = h1 - h0 > team ? (uint32_t)(h1 - h0 - team + T - 1) / T : 0u;
    Walk wr = walk_of(res, P.hd * res.cap_blocks + ((int64_t)(tiles ? h0 + team : h0) * S + mine) * 2, tiles ? tiles - 1 : 0u);
    Walk wm = wr;
    auto fetch = [&]() __attribute__((always_inline)) {   // `ahead` has the tile's bases
        ent = load_entry(res, ahead, lane);
        meta = ahead;
        step(wr, 2 * T * S);
        load_walk(wr, lay, raw);
        step(wm, 2 * T * S);
        ahead = load_meta(wm, lane);
    };
    if (prefix) {
        meta = load_meta(wm, lane);
        load_walk(wr, lay, raw);
        step(wm, 2 * T * S);
        ahead = load_meta(wm, lane);
    }
    const int parent = P.sp == A.nsp - 1 && tid < A.nodes ? A.parents[P.b * A.nodes + tid] : -2;
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

    // K or V of a tile's records into LDS, by the wave that decodes it
    auto put = [&](const Raw& d, const Meta& m, const uint4& e, uint32_t word, char* lds) {
        if (isk) {
            stage_k(d, lane, lds);
        } else {
            uint32_t vp[4][8];
            decode_v(d, vp);
            scale_v(d, word, lane, vp);
            put_v(lds, lane & 15, lane >> 4, vp);
        }
        patch_lds(isk, res, d, m, e, word, lane, s_scale[wave], lds);
    };
    if (prefix) {
        ent = load_entry(res, meta, lane);
        put(raw, meta, ent, ~0u, buf + mine * kSub);
        __builtin_amdgcn_sched_barrier(0);     // every use of the records before their reload
        fetch();
        __syncthreads();
        int t = h0, half = 0;
        for (; t + T < h1; t += T, half ^= 1) {
            put(raw, meta, ent, ~0u, buf + ((half ^ 1) * S + mine) * kSub);
            __builtin_amdgcn_sched_barrier(0);
            fetch();
            if (rows_here) {
#pragma unroll 1
                for (int u = 0; u < S; u += U) sub_attend<U>(buf + (half * S + u) * kSub, q, lane, st);
            }
            __syncthreads();
        }
        if (t + team < h1 && rows_here) {
#pragma unroll 1
            for (int u = 0; u < S; u += U) sub_attend<U>(buf + (half * S + u) * kSub, q, lane, st);
        }
        __syncthreads();
    }
    if (P.sp == A.nsp - 1) {
        if (tid == 0) s_odd = 0;
        tree_words(parent, A.nodes, s_vis, reinterpret_cast<int*>(s_buf), tid);
    }
    const int before = prefix ? h0 - seen : 0, after = prefix ? h1 : seen, edge = before + max(0, sh.end - after);
#pragma unroll 1
    for (int j = 0; j < edge; j += T) {
        const int tile = j + team < before ? seen + j + team : after + j + team - before;
        if (j + team < edge) {
            const Sub sb = sub_of<S>(A, tile, mine, P.len, P.start);
            char* lds = buf + mine * kSub;
            if (sb.word && sb.kind == 0) {
                Raw d;
                const Meta m = load_meta(res, P.hd, sb.t, A.t_prefix, lane);
                load_raw(res, P.hd, sb.t, A.t_prefix, lay, d);
                put(d, m, load_entry(res, m, lane), sb.word, lds);
            } else if (sb.word) {
                const bool draft = sb.kind == 2;
                const Rows& R = isk ? (draft ? A.dk : A.tk) : (draft ? A.dv : A.tv);
                const uint16_t* p = R.p + P.b * R.sb + P.kvh * R.sh;
                if (isk) {
                    rows_k<BF16>(p, R.st, sb.t, sb.have, lane, lds);
                } else {
                    uint32_t vp[4][8];
                    rows_v<BF16>(p, R.st, sb.t, sb.have, sb.word, lane, vp);
                    if (draft && clear_odd(vp) && lane == 0) s_odd = 1;
                    put_v(lds, lane & 15, lane >> 4, vp);
                }
            }
        }
        __syncthreads();
        if (j + team < edge && rows_here) {
#pragma unroll 1
            for (int u = 0; u < S; u++) {
                const Sub sb = sub_of<S>(A, tile, u, P.len, P.start);
                if (!sb.word) continue;
                sub_masked(buf + u * kSub, q, sb.kind == 2 ? sb.word & s_vis[node][sb.t >> 5] : sb.word, lane, st);
            }
        }
        __syncthreads();
    }

    float* dst = reinterpret_cast<float*>(s_buf) + (wave * 32 + (lane & 31)) * kMRow;
    float(*s_m)[32] = reinterpret_cast<float(*)[32]>(reinterpret_cast<float*>(s_buf) + kWaves * 32 * kMRow);
    float(*s_l)[32] = s_m + kWaves;
    const float l = st.l + __shfl_xor(st.l, 32, 64);
    if (lane < 32) {
        s_m[wave][lane] = st.m;
        s_l[wave][lane] = l;
    }
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
    join_teams<C, 32, BF16>(A, P, reinterpret_cast<const float*>(s_buf), s_m, s_l, s_vis, &s_odd, tid);
}

// Up to 16 Q rows of a kv head, Q columns of 16 a wave, tokens dealt to the waves.
template <int Q, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void k_tree_few(TreeArgs A) {
    constexpr int N = 16 * Q;                  // nodes at most: a node has a row at least
    __shared__ __align__(16) float s_buf[kWaves * 16 * Q * kMRow];
    __shared__ uint32_t s_vis[N][kVisWords];
    __shared__ int s_up[N];
    __shared__ int s_odd;                      // a draft's V has infinities or NaN
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const Place P = place_of(A, 16 * Q);
    u32x4_t* area = reinterpret_cast<u32x4_t*>(s_buf + wave * 16 * Q * kMRow);   // the wave's own until the join
    static_assert(16 * kMRow * 4 >= 8 * 64 * 16, "a tile's pairs fit it");

    const Share sh = share_of(A, P.sp);
    const int split = min(sh.end, A.np);       // prefix tiles, then rows: two loops, each with the registers it needs
    // The records of the wave's next tile are in flight during the products of this one, and
    // the bases of the tile after.  Reloads are unconditional (past the share they read the
    // last tile again), so that they land in place and nothing waits on them before their use.
    const Lay lay = lay_of(false, lane);
    KFew kr;
    Raw vr;
    Meta mk, mv, nk, nv;
    uint4 ek, ev;
    auto at = [&](int tile) { return (int64_t)min(tile, split - 1) * 32; };
    auto fetch = [&](int tile) {               // nk, nv have the tile's bases
        ek = load_entry(A.k, nk, lane);
        ev = load_entry(A.v, nv, lane);
        mk = nk;
        mv = nv;
        load_few(A.k, P.hd, at(tile), A.t_prefix, lane, kr);
        load_raw(A.v, P.hd, at(tile), A.t_prefix, lay, vr);
        nk = load_meta(A.k, P.hd, at(tile + kWaves), A.t_prefix, lane);
        nv = load_meta(A.v, P.hd, at(tile + kWaves), A.t_prefix, lane);
    };
    int tile = max(sh.first, P.first) + wave;
    const bool prefix = max(sh.first, P.first) < split;
    if (prefix) {
        mk = load_meta(A.k, P.hd, at(tile), A.t_prefix, lane);
        mv = load_meta(A.v, P.hd, at(tile), A.t_prefix, lane);
        load_few(A.k, P.hd, at(tile), A.t_prefix, lane, kr);
        load_raw(A.v, P.hd, at(tile), A.t_prefix, lay, vr);
        nk = load_meta(A.k, P.hd, at(tile + kWaves), A.t_prefix, lane);
        nv = load_meta(A.v, P.hd, at(tile + kWaves), A.t_prefix, lane);
    }
    const int parent = P.sp == A.nsp - 1 && tid < A.nodes ? A.parents[P.b * A.nodes + tid] : -2;
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
    if (prefix) {
        ek = load_entry(A.k, mk, lane);
        ev = load_entry(A.v, mv, lane);
    }
    if (P.sp == A.nsp - 1) {
        if (tid == 0) s_odd = 0;
        tree_words(parent, A.nodes, s_vis, s_up, tid);
    }
    for (; tile < split; tile += kWaves) {
        const Sub sb = sub_of<1>(A, tile, 0, P.len, P.start);
        f4_t s[Q][2];
        uint32_t vp[4][8];
#pragma unroll
        for (int x = 0; x < Q; x++) s[x][0] = s[x][1] = f4_t{0.f, 0.f, 0.f, 0.f};
        uint32_t p[8][4];                        // records 2 c + y
#pragma unroll
        for (int j = 0; j < 8; j++) {
            rec_pairs(j & 1 ? kr.a[j >> 1].y : kr.a[j >> 1].x, (kr.b[j >> 1] >> (8 * (j & 1))) & 0xffu, p[j]);
#pragma unroll
            for (int i = 0; i < 4; i++) p[j][i] = unbias(p[j][i]);
        }
        if (const uint32_t most = most_of(mk)) patch_k(A.k, kr, mk, ek, most, lane, area, p);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            mul_pairs<4>(p[j], __builtin_amdgcn_perm(0u, kr.s, j & 1 ? 0x03020302u : 0x01000100u));
#pragma unroll
            for (int x = 0; x < Q; x++)
                s[x][j & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(p[j][0], p[j][1], p[j][2], p[j][3]), q[x][j >> 1],
                                                                     s[x][j & 1], 0, 0, 0);
        }
        decode_v(vr, vp);
        if (const uint32_t most = most_of(mv)) patch_v(A.v, vr, mv, ev, most, lane, area, vp);
        scale_v(vr, sb.word, lane, vp);
        __builtin_amdgcn_sched_barrier(0);       // every use of the records before their reload
        fetch(tile + kWaves);
#pragma unroll
        for (int x = 0; x < Q; x++) few_attend(s[x], sb.word, sb.word == ~0u, vp, lane, st[x]);
    }
    if (!prefix) tile = max(sh.first, split) + wave;
    for (; tile < sh.end; tile += kWaves) {
        const Sub sb = sub_of<1>(A, tile, 0, P.len, P.start);
        if (!sb.word) continue;
        f4_t s[Q][2];
        uint32_t vp[4][8];
        const bool draft = sb.kind == 2;
        const Rows &rk = draft ? A.dk : A.tk, &rv = draft ? A.dv : A.tv;
        const uint16_t* p = rk.p + P.b * rk.sb + P.kvh * rk.sh;
        uint4 w[2][4];
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int tok = min(8 * (col >> 2) + 2 * (col & 3) + y, sb.have - 1);
                w[y][c] = *reinterpret_cast<const uint4*>(p + (sb.t + tok) * rk.st + 32 * c + 8 * g);
            }
        rows_v<BF16>(rv.p + P.b * rv.sb + P.kvh * rv.sh, rv.st, sb.t, sb.have, sb.word, lane, vp);
        if (draft && clear_odd(vp) && lane == 0) s_odd = 1;
#pragma unroll
        for (int x = 0; x < Q; x++) {
            s[x][0] = s[x][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    s[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(h8_t, BF16 ? bf_to_h(w[y][c]) : w[y][c]), q[x][c], s[x][y], 0, 0, 0);
            const uint32_t word = draft ? sb.word & s_vis[node[x]][sb.t >> 5] : sb.word;
            few_attend(s[x], word, !draft && word == ~0u, vp, lane, st[x]);
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
    join_teams<1, 16 * Q, BF16>(A, P, s_buf, s_m, s_l, s_vis, &s_odd, tid);
}

// One workgroup per row: thread (sub, dq) sums dimensions 4 dq .. + 3 of the records sub,
// sub + 8, .. (their loads go out together), then the eight sums are joined in order.
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs A, int bf16) {
    constexpr int kUp = 8;                     // records in flight per thread
    __shared__ __align__(16) f4_t s_o[8][32];
    __shared__ float s_m[8], s_l[8];
    const int dq = threadIdx.x & 31, sub = threadIdx.x >> 5;
    const int64_t hd = blockIdx.x / (uint32_t)A.rows;
    const int r = (int)(blockIdx.x % (uint32_t)A.rows);
    const float* rec = A.rec + (hd * A.nsp * A.rows + r) * kRecF;
    const int64_t step = (int64_t)A.rows * kRecF;
    const float tail_l = rec[(A.nsp - 1) * step + 1];
    float m = -INFINITY, l = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = sub; p0 < A.nsp; p0 += 8 * kUp) {
        float2 ml[kUp];
        f4_t v[kUp];
#pragma unroll
        for (int k = 0; k < kUp; k++) {
            const float* x = rec + min(p0 + 8 * k, A.nsp - 1) * step;
            ml[k] = *reinterpret_cast<const float2*>(x);
            v[k] = *reinterpret_cast<const f4_t*>(x + 4 + 4 * dq);
        }
        float M = m;
#pragma unroll
        for (int k = 0; k < kUp; k++) M = p0 + 8 * k < A.nsp ? fmaxf(M, ml[k].x) : M;
        const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M);
        o *= f0;
        l *= f0;
#pragma unroll
        for (int k = 0; k < kUp; k++) {
            if (p0 + 8 * k >= A.nsp) continue;
            const float f = ml[k].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[k].x - M);
            l = __builtin_fmaf(ml[k].y, f, l);
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(v[k][c], f, o[c]);
        }
        m = M;
    }
    s_o[sub][dq] = o;
    if (dq == 0) {
        s_m[sub] = m;
        s_l[sub] = l;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; k++) M = fmaxf(M, s_m[k]);
    float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float f = s_m[k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[k] - M);
        const float2 v = reinterpret_cast<const float2*>(s_o[k])[lane];
        L = __builtin_fmaf(s_l[k], f, L);
        x = __builtin_fmaf(v.x, f, x);
        y = __builtin_fmaf(v.y, f, y);
    }
    const bool empty = tail_l == kEmpty;
    const float inv = 1.f / L;
    out_pair(A, bf16 != 0, hd / A.heads, hd % A.heads, r, 2 * lane, empty ? 0.f : x * inv, empty ? 0.f : y * inv);
}

// ------------------------------------------------------------------- plan --

struct Plan {
    int c, rb, np, nt, nd, nsp, per;
};

// Waves of a team (c): as many 32-row columns as there are rows, eight at most (their O is
// 64 registers each), so that a tile is decoded once for all of them.  Where little is to
// be read, decoding it for two halves of the rows on twice the CUs is faster: a round is
// 128 tokens in all three forms, and takes 5 us (c = 8, beside 16 us before and after the
// rounds), 3.7 us (4, beside 11 us).  Measured, one sequence of 8 heads with a tail of
// 100, 256 rows a head: 8192 tokens (2 rounds a CU with c = 8) 38.0 us with c = 8, 35.8
// with 4; 16384 tokens 47.7 / 47.3; 32768 tokens (8 rounds) 67 / 75.  128 rows: 4096
// tokens (1 round with c = 4) 25.6 us with c = 4, 23.7 with 2; 16384 (4 rounds) 34.8 / 38.6.
constexpr int64_t kRounds8 = 3, kRounds4 = 2;
// Costs of the choice of splits, in units of half a round: a round over whole prefix
// tiles, one over the others (the tail's, the draft's, the prefix's last), and a
// workgroup's prologue and join.  A split's share is whole rounds of its teams' tiles; of
// the splits whose longest CU takes the least the fewest (records are written and read
// again).  The last one has the draft and whatever the equal shares leave: a share more
// for the draft alone is often the best (one head of 16384 tokens, 64 rows: 17.6 us;
// 20.1 with the draft beside a full share).
constexpr uint32_t kHotCost = 2, kEdgeCost = 2, kFixedCost = 3;
bool plan(int64_t n_seq, int64_t heads, int64_t nodes, int64_t group, int64_t t_prefix, int64_t tail_cap, Plan* p) {
    if (n_seq < 1 || heads < 1 || nodes < 1 || nodes > kMaxNodes || group < 1 || group > 16 || t_prefix < 0 ||
        t_prefix % kRB || tail_cap < 0 || t_prefix > INT_MAX / 2 || tail_cap > INT_MAX / 4)
        return false;
    const int64_t rows = nodes * group;
    p->c = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;   // 1: k_tree_few
    const auto blocks = [=](int c) { return (rows + 32 * c - 1) / (32 * c); };
    const auto rounds_a_cu = [=](int c) { return n_seq * heads * blocks(c) * ((t_prefix + tail_cap + 127) / 128) / 256; };
    if (n_seq > INT_MAX / heads) return false;
    if (p->c == 8 && rounds_a_cu(8) <= kRounds8) p->c = 4;
    if (p->c == 4 && rounds_a_cu(4) <= kRounds4) p->c = 2;
    const int64_t s = p->c > 1 ? p->c / 2 : 1, tt = 32 * s;
    p->rb = (int)blocks(p->c);
    p->np = (int)((t_prefix + tt - 1) / tt);
    p->nt = (int)((tail_cap + tt - 1) / tt);
    p->nd = (int)((nodes + tt - 1) / tt);
    const int64_t base = n_seq * heads * p->rb;
    if (base > INT_MAX / 256) return false;
    const int lg = p->c > 1 ? (p->c == 8 ? 0 : p->c == 4 ? 1 : 2) : 3;   // teams = 1 << lg
    const auto rounds_of = [lg](uint32_t n) { return (n + (1u << lg) - 1) >> lg; };
    const uint32_t np = (uint32_t)p->np, cache = np + (uint32_t)p->nt, tiles = cache + (uint32_t)p->nd, whole = (uint32_t)(t_prefix / tt);
    int64_t best = -1;
    const uint32_t most = (uint32_t)std::min<int64_t>(256, std::max<int64_t>(4, 512 / base));
    for (uint32_t n = 1; n <= most && (n == 1 || n <= tiles); n++) {
        // n splits share the prefix, the cache or all tiles in equal parts; the last takes what is left
        const uint32_t of[3] = {np, cache, tiles};
        uint32_t was = 0;
        for (uint32_t x : of) {
            const uint32_t rounds = std::max(rounds_of((x + n - 1) / n), 1u);
            if (rounds == was) continue;
            was = rounds;
            const uint32_t first = std::min<uint64_t>((uint64_t)(n - 1) * rounds << lg, cache), hot = whole > first ? whole - first : 0u;
            const uint32_t last = kHotCost * rounds_of(hot) + kEdgeCost * rounds_of(tiles - first - hot);
            const int64_t cost = (base * n + 255) / 256 * (int64_t)(kHotCost * rounds + kFixedCost) +
                                 (last > kHotCost * rounds ? last - kHotCost * rounds : 0u);
            if (best < 0 || cost < best) {
                best = cost;
                p->nsp = (int)n;
                p->per = (int)(rounds << lg);
            }
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
    if (c == 8) hipLaunchKernelGGL((k_tree_many<8, BF16>), g, wg, 0, s, A);
    else if (c == 4) hipLaunchKernelGGL((k_tree_many<4, BF16>), g, wg, 0, s, A);
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
                               void *d_work, int64_t work_bytes, const lq_rows *out, hipStream_t s) {
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
    if (work_bytes < lq_tree_attn_workspace(n_seq, heads, n_nodes, group, t_prefix, tail_cap) || ((uintptr_t)d_work & 15))
        return LQ_ERR_ARG;
    TreeArgs A{};
    if (t_prefix > 0) {
        A.k = *k;
        A.v = *v;
        // an empty exception list is read at its first entry and the value not used
        if (!A.k.exc || A.k.exc_cap == 0) A.k.exc = reinterpret_cast<int16_t*>(A.k.a);
        if (!A.v.exc || A.v.exc_cap == 0) A.v.exc = reinterpret_cast<int16_t*>(A.v.a);
    }
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
    A.per = p.per;
    A.tiles = p.np + p.nt + p.nd;
    A.rec = static_cast<float*>(d_work);
    const int64_t grid = k->n_heads * p.nsp * p.rb;
    if (dtype == LQ_BF16) tree_launch<true>(A, p.c, grid, s);
    else tree_launch<false>(A, p.c, grid, s);
    if (p.nsp > 1) {
        hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)(k->n_heads * A.rows)), dim3(256), 0, s, A, dtype == LQ_BF16);
    }
    return launch_status();
}

}  // extern "C"
