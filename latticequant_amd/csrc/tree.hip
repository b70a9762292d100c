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
// One workgroup of eight waves per (kv head, block of 32 C rows, split of the
// tokens): C waves (a team) hold 32 rows each and share their tokens, 8 / C teams
// take the split's tiles in turn.  A tile is decoded once into LDS by its team
// (K as rows, V with its dimensions as rows) and read by all of it:
//   S^T = K Q^T     8 MFMA 32x32x16 per 32 tokens: lane column n is row n of the
//                   wave, so max and sum of a row are in-lane but for one swap of
//                   the wave's halves
//   O^T += V^T P^T  8 MFMA.  K's row m of a tile is token
//                   16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4: then the
//                   scores a lane holds are those of tokens 16 s + 8 g .. + 7, which
//                   is the B operand of step s as it stands: P never leaves its lane.
// V's LDS row 16 i + n is dimension 8 n + i, the order in which a lane has the
// eight dimensions of a decoded vector.
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

__device__ __forceinline__ uint32_t pair_h(float a, float b) {
    const h2_t r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
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

// Addresses of 32 prefix tokens from t on; the second block of the last tile may lie
// past the prefix: the last block is read in its place (its tokens are outside the word).
struct Blocks {
    int64_t rb0, tb0;
    uint32_t d;      // 1, or 0 where the second block is clamped
};
__device__ __forceinline__ Blocks blocks_of(const lq_resident& r, int64_t hd, int64_t t, int64_t T) {
    Blocks b;
    b.tb0 = t;
    b.d = t + kRB < T ? 1u : 0u;
    b.rb0 = hd * r.cap_blocks + t / kRB;
    return b;
}

__device__ void prefix_k(const lq_resident& r, int64_t hd, int64_t t, int64_t T, int lane, char* lds) {
    const Blocks B = blocks_of(r, hd, t, T);
    uint32_t a[2][4], b[2][4], s[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int64_t rb = B.rb0 + (x ? B.d : 0u);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            a[x][c] = r.a[rb * 256 + c * 64 + lane];
            b[x][c] = r.b[rb * 256 + c * 64 + lane];
        }
        s[x] = r.scale[hd * r.cap_blocks * kRB + B.tb0 + (x ? B.d * kRB : 0u) + (lane & 15)];
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int64_t rb = B.rb0 + (x ? B.d : 0u);
        const uint32_t count = __builtin_amdgcn_readfirstlane(r.meta[rb * 4 + 3]);
        int64_t base = __builtin_amdgcn_readfirstlane(r.meta[rb * 4 + 2]);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t p[4];
            rec_pairs(a[x][c], b[x][c], p);
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = unbias(p[i]);
            if (count) {
                const uint64_t m = r.mask[rb * 4 + c];
                const int64_t idx = base + __builtin_popcountll(m & ((1ull << lane) - 1ull));
                if (((m >> lane) & 1ull) && idx < r.exc_cap) {
                    int v[8];
                    exc_load(r.exc, idx, v);
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] = pair_from_i16(v[2 * i], v[2 * i + 1]);
                }
                base += __builtin_popcountll(m);
            }
            mul_pairs<4>(p, s[x] * 0x00010001u);
            put_k(lds, 16 * x + (lane & 15), 4 * c + (lane >> 4), make_uint4(p[0], p[1], p[2], p[3]));
        }
    }
}

__device__ void prefix_v(const lq_resident& r, int64_t hd, int64_t t, int64_t T, uint32_t word, int lane, char* lds) {
    const Blocks B = blocks_of(r, hd, t, T);
    const int n = lane & 15, k8 = lane >> 4;
    const int64_t rb = B.rb0 + ((k8 >> 1) ? B.d : 0u);
    const int64_t r0 = rb * 256 + (n >> 2) * 64 + 16 * (n & 3) + 8 * (k8 & 1);
    const uint4 a0 = reinterpret_cast<const uint4*>(r.a + r0)[0], a1 = reinterpret_cast<const uint4*>(r.a + r0)[1];
    const uint2 bw = *reinterpret_cast<const uint2*>(r.b + r0);
    const uint4 sc = *reinterpret_cast<const uint4*>(r.scale + hd * r.cap_blocks * kRB + B.tb0 +
                                                     ((k8 >> 1) ? B.d * kRB : 0u) + 8 * (k8 & 1));
    const uint32_t aw[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
    uint32_t vp[4][8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t w = k < 2 ? bw.x : bw.y;
        rec_pairs_tok(aw[2 * k], w >> (16 * (k & 1)), aw[2 * k + 1], w >> (16 * (k & 1) + 8), vp[k]);
#pragma unroll
        for (int i = 0; i < 8; i++) vp[k][i] = unbias(vp[k][i]);
    }
    if (r.meta[rb * 4 + 3]) {
        int64_t base = r.meta[rb * 4 + 2];
        for (int c = 0; c < (n >> 2); c++) base += __builtin_popcountll(r.mask[rb * 4 + c]);
        const uint64_t m = r.mask[rb * 4 + (n >> 2)];
        const int s0 = 16 * (n & 3) + 8 * (k8 & 1);
        base += __builtin_popcountll(m & ((1ull << s0) - 1ull));
        const uint32_t own = (uint32_t)(m >> s0) & 0xffu;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const int64_t idx = base + __builtin_popcount(own & ((1u << q) - 1u));
            if (((own >> q) & 1u) && idx < r.exc_cap) {
                int v[8];
                exc_load(r.exc, idx, v);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    h2_t h = __builtin_bit_cast(h2_t, vp[q >> 1][i]);
                    h[q & 1] = (_Float16)((float)v[i] * 0.5f);
                    vp[q >> 1][i] = __builtin_bit_cast(uint32_t, h);
                }
            }
        }
    }
    const uint32_t sw[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
    for (int k = 0; k < 4; k++) mul_pairs<8>(vp[k], sw[k]);
    if (word != ~0u) clear_v(word, k8, vp);
    put_v(lds, n, k8, vp);
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

// returns whether one of the values is an infinity or a NaN
template <bool BF16>
__device__ bool rows_v(const Rows& R, int64_t b, int64_t h, int64_t t, uint32_t word, int lane, char* lds) {
    const uint16_t* p = R.p + b * R.sb + h * R.sh;
    const int n = lane & 15, k8 = lane >> 4;
    uint32_t vp[4][8];
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
    put_v(lds, n, k8, vp);
    return __any(bad != 0u);
}

// ---------------------------------------------------------- 32 x 32 of it --

struct RowState {
    float m, l;      // running maximum (base 2), the lane's part of the sum
    f16_t o[4];      // O^T: column lane % 32, row of MFMA dt: V row 32 dt + 8 (i / 4) + 4 (lane / 32) + i % 4
};

// token of score register i of a lane, without its half's 8 (lane / 32)
constexpr int tok_of(int i) { return 16 * (i >> 3) + 4 * ((i >> 2) & 1) + (i & 3); }

__device__ __forceinline__ float halves_max(float v) {
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// One subtile for the wave's 32 rows: word has the visible tokens of the lane's
// row; every: all of them, for every lane.
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
    if (!odd) {
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

template <int C, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void k_tree_attn(TreeArgs A) {
    constexpr int S = C > 1 ? C / 2 : 1;       // subtiles of a tile
    constexpr int T = kWaves / C;              // teams
    constexpr int kStage = T * S * kSub, kMerge = kWaves * 32 * kMRow * 4;
    __shared__ __align__(16) char s_buf[kStage > kMerge ? kStage : kMerge];
    __shared__ uint32_t s_vis[kMaxNodes][kVisWords];
    __shared__ int s_up[kMaxNodes];
    __shared__ int s_bad[T][S];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int team = wave / C, ct = wave % C;
    int64_t bid = blockIdx.x;
    const int rblk = (int)(bid % A.rb);
    bid /= A.rb;
    const int sp = (int)(bid % A.nsp);
    const int64_t hd = bid / A.nsp;            // resident head: sequence * heads + kv head
    const int64_t b = hd / A.heads, kvh = hd % A.heads;
    const int row0 = rblk * 32 * C;
    const int64_t len = A.tail_cap ? (A.tail_len ? min((int64_t)max(A.tail_len[b], 0), A.tail_cap) : A.tail_cap) : 0;
    const int64_t start = A.start ? A.start[b] : 0;
    const bool last = sp == A.nsp - 1;
    if (last) tree_words(A.parents + b * A.nodes, A.nodes, s_vis, s_up, tid);

    // the wave's rows: column lane % 32
    const int r = row0 + 32 * ct + (lane & 31);
    const int node = r < A.rows ? r / A.group : 0;
    h8_t q[8];
#pragma unroll
    for (int c = 0; c < 8; c++) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (r < A.rows)
            w = load_row8<BF16>(A.q.p + b * A.q.sb + (kvh * A.group + r % A.group) * A.q.sh + (int64_t)node * A.q.st +
                                16 * c + 8 * (lane >> 5));
        q[c] = __builtin_bit_cast(h8_t, w);
    }
    RowState st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) st.o[d][i] = 0.f;

    // split sp takes `per` of the tiles; the draft's all fall to the last
    const int per = (A.tiles + A.nsp - 1) / A.nsp, cache = A.np + A.nt;
    const int first = min(sp * per, cache), end = last ? A.tiles : min((sp + 1) * per, cache);
    char* buf = s_buf + team * S * kSub;
    for (int t0 = first; t0 < end; t0 += T) {
        const int tile = t0 + team;
        if (tile < end) {
#pragma unroll
            for (int u = 0; u < S; u++) {
                const Sub sb = sub_of<S>(A, tile, u, len, start);
                if (!sb.word) continue;
                char* lds = buf + u * kSub;
                if (C == 1 || ct == u) {
                    if (sb.kind == 0) prefix_k(A.k, hd, sb.t, A.t_prefix, lane, lds);
                    else rows_k<BF16>(sb.kind == 1 ? A.tk : A.dk, b, kvh, sb.t, sb.word, lane, lds);
                }
                if (C == 1 || ct == S + u) {
                    if (sb.kind == 0) {
                        prefix_v(A.v, hd, sb.t, A.t_prefix, sb.word, lane, lds);
                    } else {
                        const bool bad = rows_v<BF16>(sb.kind == 1 ? A.tv : A.dv, b, kvh, sb.t, sb.word, lane, lds);
                        if (lane == 0) s_bad[team][u] = bad;
                    }
                }
            }
        }
        __syncthreads();
        if (tile < end && row0 + 32 * ct < A.rows) {
#pragma unroll
            for (int u = 0; u < S; u++) {
                const Sub sb = sub_of<S>(A, tile, u, len, start);
                if (!sb.word) continue;
                uint32_t w = sb.word;
                if (sb.kind == 2) w &= s_vis[node][sb.t >> 5];
                const bool odd = sb.kind == 2 && __builtin_amdgcn_readfirstlane(s_bad[team][u]);
                sub_attend(buf + u * kSub, q, w, sb.kind != 2 && sb.word == ~0u, odd, lane, st);
            }
        }
        __syncthreads();
    }

    // ---- the teams' (m, l, O) of each row joined through LDS
    {
        const float l = st.l + __shfl_xor(st.l, 32, 64);
        if (lane < 32) {
            s_m[wave][lane] = st.m;
            s_l[wave][lane] = l;
        }
        float* dst = reinterpret_cast<float*>(s_buf) + (wave * 32 + (lane & 31)) * kMRow;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {      // vector 8 j + 4 (lane / 32) + i: dimensions 8 n + 2 d + h
                float* x = dst + 8 * (8 * j + 4 * (lane >> 5) + i);
                *reinterpret_cast<f4_t*>(x) = f4_t{st.o[0][4 * j + i], st.o[0][8 + 4 * j + i], st.o[1][4 * j + i],
                                                   st.o[1][8 + 4 * j + i]};
                *reinterpret_cast<f4_t*>(x + 4) = f4_t{st.o[2][4 * j + i], st.o[2][8 + 4 * j + i], st.o[3][4 * j + i],
                                                       st.o[3][8 + 4 * j + i]};
            }
    }
    __syncthreads();
    const float* mb = reinterpret_cast<const float*>(s_buf);
    for (int idx = tid; idx < 32 * C * (kHd / 2); idx += kWaves * 64) {
        const int lr = idx / (kHd / 2), d = 2 * (idx % (kHd / 2));
        const int rr = row0 + lr;
        if (rr >= A.rows) break;               // idx grows with the row
        const int w0 = lr >> 5, c = lr & 31;
        float M = -INFINITY;
#pragma unroll
        for (int t = 0; t < T; t++) M = fmaxf(M, s_m[t * C + w0][c]);
        float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const int w = t * C + w0;
            const float f = s_m[w][c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w][c] - M);
            L += s_l[w][c] * f;
            x += mb[(w * 32 + c) * kMRow + d] * f;
            y += mb[(w * 32 + c) * kMRow + d + 1] * f;
        }
        const int nd = rr / A.group;
        const bool empty = last && !((s_vis[nd][nd >> 5] >> (nd & 31)) & 1u);
        if (A.nsp == 1) {
            const float inv = 1.f / L;
            out_pair(A, BF16, b, kvh, rr, d, empty ? 0.f : x * inv, empty ? 0.f : y * inv);
        } else {
            float* rec = A.rec + ((hd * A.nsp + sp) * A.rows + rr) * kRecF;
            *reinterpret_cast<float2*>(rec + 4 + d) = make_float2(x, y);
            if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(M, empty ? kEmpty : L);
        }
    }
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
    p->c = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
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

template <int C>
void tree_launch(const TreeArgs& A, bool bf16, int64_t grid, hipStream_t s) {
    if (bf16) hipLaunchKernelGGL((k_tree_attn<C, true>), dim3((unsigned)grid), dim3(kWaves * 64), 0, s, A);
    else hipLaunchKernelGGL((k_tree_attn<C, false>), dim3((unsigned)grid), dim3(kWaves * 64), 0, s, A);
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
    if (p.c == 1) tree_launch<1>(A, dtype == LQ_BF16, grid, s);
    else if (p.c == 2) tree_launch<2>(A, dtype == LQ_BF16, grid, s);
    else tree_launch<4>(A, dtype == LQ_BF16, grid, s);
    if (p.nsp > 1) {
        const int64_t n = k->n_heads * A.rows;
        hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s, A, n, dtype == LQ_BF16);
    }
    return launch_status();
}

}  // extern "C"
