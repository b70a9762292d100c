// One new token of each of many sequences over a pool of resident pages, for gfx950,
// with the softmax weight of every page, and the choice of pages by that weight.
//
// A page is one resident block (16 tokens) of every kv head of the pool; sequence b has
// n_pages[b] of them, by number and in order in its row of the table, and tail_len[b]
// rows behind them.  With z = q . k log2(e) / sqrt(128) a row (query head) has
//   o = sum_t 2^(z_t - m) v_t / sum_t 2^(z_t - m),   m = max_t z_t,
// taken in one pass (m raised lazily, as in the tree's kernels), and page j the weight
//   w_j = sum over the kv heads' rows of 2^(z(row, j) - lse(row)),
// z(row, j) the logarithm of the page's own sum, lse that of all.
//
// The work is the list of all 32-token tiles, sequence by sequence, head by head, the
// pages' before the tail's.  Its length is known on the device only: every workgroup sums
// the sequences' tiles and takes an equal share of the list, every wave an equal part of
// that, so lengths of any mix load the chip evenly.  A (sequence, head) that lies within
// a wave is written out by it; the pieces of one that several waves share are joined in
// LDS, those that several workgroups share by k_paged_join, in the order of the list.  (The
// last of the workgroups joining them itself, by a counter per unit, was no faster: its
// device-scope stores, release and acquire took the 4 to 5 us of the second launch with 136
// tiles, and 9 us more than it with 8200.)
//
// Long ones are bound by instructions and memory alike: 520 vector instructions a tile (decode
// of K and V about 345, K's exceptions through LDS and back 60, softmax of a lane's two
// tokens and both products' rest 115) at two waves a SIMD, one tile in flight beside the
// one that is worked on; 2 sequences of 131072 tokens, 8 heads, 4 rows, 8 % of K's vectors
// exceptions: 87 to 92 us, 3.9 to 4.1 TB/s (of a form of 480 instructions, 83 to 87: three waves
// a SIMD 105, two tiles in flight 139, both spill).
// Short ones by latency (32 sequences up to 2048 tokens: two fifths of the waves' cycles they
// wait, a third they issue): lengths, table, records and exceptions are loaded in turn, and a
// tile takes a lone wave 4200 cycles; 1 sequence of 500 tokens 11.0 us.
#include <climits>
#include <cmath>
#include <type_traits>

#include "lq_device.h"
#include "lq_few.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

constexpr int kWaves = 4;                      // of a workgroup that takes a share
constexpr int kWholeWaves = 8;                 // of one that takes a unit, where each has a compute unit
constexpr int kGroups = 512;                   // workgroups at most
// Where no (sequence, head) can have more than kWhole tiles and all fit on the chip at once, a
// workgroup takes one as a whole, of eight waves where each finds a compute unit, and there is
// no second launch.  1 / 8 / 32 sequences of 8 heads, replayed from a graph, against equal
// shares: 4 tiles 5.9 / 6.1 / 6.2 us (8.9 / 9.8 / 10.0), 20 tiles 9.5 / 10.2 / 10.9 (11.1 / 13.0 /
// 16.7), 32 tiles 12.6 / 13.6 / 15.1 (11.1 / 14.0 / 20.7), the host's 3 us for a launch not
// counted; 48 tiles 16.3 / 17.7 / 19.2 (11.5 / 15.4 / 24.2), and lengths may differ.  64
// sequences, with four waves so that all are there at once: 2 / 16 / 32 tiles 6.0 / 15.0 / 22.8
// (shares 8.7 / 19.7 / 26.9, eight waves 10.0 / 19.7 / 27.7).  A kernel of its own, without what
// finds shares: code that is only branched around cost 0.9 us (with 17 tiles).
constexpr int kWhole = 32;
// A unit's first tile waits for its page numbers, records and exceptions in turn and its tail
// for its rows, which took about two tiles' time: the list has two places for that before each
// unit's tiles.  32 sequences up to 2048 tokens / 64 up to 8192 with weights, a call: one place
// 23.2 / 119.0 us, two 23.3 / 116.9, four 24.1 / 117.3 (without any the kernel took 2.5 / 8 more).
constexpr int kAhead = 2;
constexpr int kMRow = kHd + 4;                 // floats of a piece's row in LDS: o[128], m, l, l32
constexpr int kRecF = 4 + kHd;                 // floats of a record's row: m, l, l32, unused, o[128]
constexpr int kPatch = 8 * 64 * 16;            // bytes of a wave's area for exceptions

struct Rows {
    const uint16_t* p;
    int64_t sb, sh, st;
};

// A unit: the sequence's number and the head's (of at most 65535 each), none: ~0.
__device__ __forceinline__ uint32_t unit_of(int b, int h) { return (uint32_t)b << 16 | (uint32_t)h; }
struct Desc {                                  // the unit that a workgroup leaves unfinished
    uint32_t unit;
    int32_t more;                              // the workgroups that follow it there
};

struct PagedArgs {
    lq_pages k, v;
    const int32_t* pages;
    const int32_t* n_pages;
    const int32_t* tail_len;
    int64_t width, tail_cap;
    Rows q, tk, tv;
    uint16_t* out;
    int64_t ob, oh;
    int n_seq, heads, group, per;              // per: sequences of a lane's sum
    int ahead;                                 // places of the list that a unit has before its tiles'
    float* rec;                                // [2 workgroup + (0: of an earlier one's, 1: begun here)][row][kRecF]
    Desc* desc;
    float* lse;                                // [unit][row]: m + log2(l32), with the weights' factor 2^kPShift
    float* z;                                  // [unit][page][row]
};

struct Len {
    int pages, tail, tiles, page_tiles;
    uint32_t places;                           // of the list, for a head
};
__device__ __forceinline__ Len len_of(const PagedArgs& A, int b) {
    Len l;
    l.pages = min(max(A.n_pages[b], 0), (int)A.width);
    l.tail = A.tail_cap ? (A.tail_len ? min(max(A.tail_len[b], 0), (int)A.tail_cap) : (int)A.tail_cap) : 0;
    l.page_tiles = (l.pages + 1) >> 1;
    l.tiles = l.page_tiles + ((l.tail + 31) >> 5);
    l.places = l.tiles ? (uint32_t)(l.tiles + A.ahead) : 0u;
    return l;
}

// Bytes from a plane's base to a block: 32 bits where the plane is shorter than 4 GiB.
template <bool BIG>
struct Off {
    typedef uint32_t type;
};
template <>
struct Off<true> {
    typedef uint64_t type;
};
template <typename T, typename O>
__device__ __forceinline__ T at(const void* base, O bytes) {
    return *reinterpret_cast<const T*>(static_cast<const char*>(base) + bytes);
}

// Records of a tile's blocks b0 and b1: of K, pairs of tokens 8 g + 2 i, + 1 (lane % 16 =
// 4 g + i) of vectors 4 c + lane / 16; of V, vector lane % 16 of tokens 8 (lane / 16) .. + 7.
// A copy that is made here: where a register's next value is being loaded, the compiler
// would copy the loaded one at the loop's end instead, and wait for it there.
__device__ __forceinline__ uint32_t copied(uint32_t x) {
    uint32_t y;
    asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
    return y;
}
struct Recs {
    uint2 ka[4];
    uint32_t kb[4];
    uint4 va[2];
    uint2 vb;
    uint32_t vs[4], ks[4];                     // scales of V and K of the tokens that the lane weighs, pairs
    uint32_t kp;                               // of K where the records lie, where they are multiplied there
};
// The lanes of a quarter (16) hold the scores of eight tokens of 16 rows, but a group has
// mostly fewer: with NR row slots lane r + NR a of a quarter weighs row r's tokens
// (NR / 2) a .. + NR / 2 - 1.  Pairs of tokens a lane weighs, and their scales:
template <int NR>
constexpr int kPairs = NR / 4;
template <int NR, typename O>
__device__ __forceinline__ void load_scales(const uint16_t* scale, O at_block, uint32_t lane, uint32_t s[4]) {
    const O from = at_block + (lane & 16) + (lane & 15) / NR * (NR / 4) * 4;
    if constexpr (NR == 16) {
        const uint4 w = at<uint4>(scale, from);
        s[0] = w.x; s[1] = w.y; s[2] = w.z; s[3] = w.w;
    } else if constexpr (NR == 8) {
        const uint2 w = at<uint2>(scale, from);
        s[0] = w.x; s[1] = w.y;
    } else {
        s[0] = at<uint32_t>(scale, from);
    }
}
struct Meta2 {
    uint32_t base, count;                      // exceptions of block lane / 32
};
template <bool BIG, bool ROUND, int NR>
__device__ __forceinline__ void load_k(const PagedArgs& A, uint32_t b0, uint32_t b1, uint32_t lane, Recs& d) {
    typedef typename Off<BIG>::type O;
    const uint32_t row = lane & 15, blk = row & 8 ? b1 : b0, tok = 8 * ((row >> 2) & 1) + 2 * (row & 3), rec = 16 * (lane >> 4) + tok;
    const O a = (O)blk * 1024 + rec * 4, b = (O)blk * 256 + rec;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        d.ka[c] = at<uint2>(A.k.r.a, a + 256 * c);
        d.kb[c] = at<uint16_t>(A.k.r.b, b + 64 * c);
    }
    if constexpr (ROUND) d.kp = at<uint32_t>(A.k.r.scale, (O)blk * 32 + tok * 2);
    else load_scales<NR>(A.k.r.scale, (O)(lane & 32 ? b1 : b0) * 32, lane, d.ks);
}
template <bool BIG, int NR>
__device__ __forceinline__ void load_v(const PagedArgs& A, uint32_t b0, uint32_t b1, uint32_t lane, Recs& d) {
    typedef typename Off<BIG>::type O;
    const uint32_t blk = lane & 32 ? b1 : b0, rec = 16 * (lane & 15) + (lane & 16 ? 8 : 0);
    const O a = (O)blk * 1024 + rec * 4;
    d.va[0] = at<uint4>(A.v.r.a, a);
    d.va[1] = at<uint4>(A.v.r.a, a + 16);
    d.vb = at<uint2>(A.v.r.b, (O)blk * 256 + rec);
    load_scales<NR>(A.v.r.scale, (O)blk * 32, lane, d.vs);
}
template <bool BIG>
__device__ __forceinline__ Meta2 load_meta(const lq_pages& p, uint32_t b0, uint32_t b1, uint32_t lane) {
    typedef typename Off<BIG>::type O;
    const uint2 w = at<uint2>(p.r.meta, (O)(lane & 32 ? b1 : b0) * 16 + 8);
    return {w.x, w.y};
}
// The first 32 exceptions of each block, one a lane, with the number of its record.
struct Entry {
    uint4 v;
    uint32_t rec;
};
template <bool BIG>
__device__ __forceinline__ Entry load_entry(const lq_pages& p, const Meta2& m, uint32_t e) {
    typedef typename Off<BIG>::type O;
    const uint32_t i = m.base + e, from = e < m.count && i < (uint32_t)p.r.exc_cap ? i : 0u;
    return {at<uint4>(p.r.exc, (O)from * 16), at<uint8_t>(p.rec, from)};
}
__device__ __forceinline__ uint32_t most_of(const Meta2& m) {   // wave-uniform
    return max((uint32_t)__builtin_amdgcn_readlane((int)m.count, 0), (uint32_t)__builtin_amdgcn_readlane((int)m.count, 32));
}
// put(rec, v): the lane's entry over record rec of block lane / 32, for all of a tile, 32 of
// a block at a time (in the place of one that the list had no room for stands the zero vector)
template <bool BIG, typename P>
__device__ __forceinline__ void each_entry(const lq_pages& p, const Meta2& m, Entry e, uint32_t most, int lane, P put) {
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < most; r0 += 32) {
        const uint32_t k = r0 + (lane & 31);
        if (r0) e = load_entry<BIG>(p, m, k);
        if (k < m.count && m.base + k < (uint32_t)p.r.exc_cap) put(e.rec, e.v);
    }
}

// K's records without their bias: as a pair of fp16 numbers 2^-24 w, w = 2 c + 32, whole and
// below 64 for a record.  What is multiplied by them needs neither the 32 taken off nor the
// scale: both go into the other operand's sum and into the product (see attend below).
template <int SH>   // b's byte from bit SH on
__device__ __forceinline__ void raw_pairs(uint32_t a, uint32_t b, uint32_t p[4]) {
    const uint32_t kc = __builtin_amdgcn_perm(0u, a, 0x0c000c00u) & 0x00010001u;
    p[0] = (a & kFieldMask) | kc;
    p[1] = ((a >> 5) & kFieldMask) | kc;
    p[2] = ((a >> 10) & kFieldMask) | kc;
    const uint32_t u6 = (b >> SH) & 31u, c7h = ((b >> (SH + 5)) & 7u) | ((a >> 13) & 8u);
    const uint32_t par = ((uint32_t)__builtin_popcount(a & kLsbMask) + u6) & 1u;
    p[3] = kc | (u6 << 1) | (((c7h << 1) | par) << 17);
}
// V's as coordinates c.  (As 2^-24 w, with 2^-19 sum P taken off the sums, V cost 32 instructions a
// tile less, 0.5 to 3 us of the cases; but the products' unit drops what lies 2^-24 below its
// largest term, taking a subnormal number's exponent for 2^-14 where w = 32 is 2^-19: beside
// a token of nearly all the weight the 31 others lost up to 2^-15 of a scale each, and the taking
// off is as exact as w, not as c.)
template <int SH, int K>   // both bytes, from bits SH and SH + 8 on, into each dimension's pair K
__device__ __forceinline__ void pairs_tok(uint32_t a0, uint32_t a1, uint32_t b, u32x4_t p[8]) {
    const uint32_t lo = __builtin_amdgcn_perm(a1, a0, 0x05040100u);
    const uint32_t hi = __builtin_amdgcn_perm(a1, a0, 0x07060302u);
    const uint32_t kc = 0x60006000u | (lo & 0x00010001u);   // 512 and the coset's half
    p[0][K] = unbias((lo & kFieldMask) | kc);
    p[2][K] = unbias(((lo >> 5) & kFieldMask) | kc);
    p[4][K] = unbias(((lo >> 10) & kFieldMask) | kc);
    p[1][K] = unbias((hi & kFieldMask) | kc);
    p[3][K] = unbias(((hi >> 5) & kFieldMask) | kc);
    p[5][K] = unbias(((hi >> 10) & kFieldMask) | kc);
    const uint32_t u0 = (b >> SH) & 31u, u1 = (b >> (SH + 8)) & 31u;
    const uint32_t h0 = ((b >> (SH + 5)) & 7u) | ((a0 >> 13) & 8u);
    const uint32_t h1 = ((b >> (SH + 13)) & 7u) | ((a1 >> 13) & 8u);
    const uint32_t q0 = ((uint32_t)__builtin_popcount(a0 & kLsbMask) + u0) & 1u;
    const uint32_t q1 = ((uint32_t)__builtin_popcount(a1 & kLsbMask) + u1) & 1u;
    p[6][K] = unbias(kc | (u0 << 1) | (u1 << 17));
    p[7][K] = unbias(kc | (((h0 << 1) | q0) << 1) | (((h1 << 1) | q1) << 17));
}
// an entry of K's eight values 2c so (beyond 2048 they lose bits, as fp16 does)
__device__ __forceinline__ void raw_entry(const uint4& w, uint32_t p[4]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    const h2_t tiny = __builtin_bit_cast(h2_t, 0x00010001u), bias = __builtin_bit_cast(h2_t, 0x00200020u);   // 2^-24, 2^-19
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2_t h = {(_Float16)(int16_t)(x[i] & 0xffffu), (_Float16)(int16_t)(x[i] >> 16)};
        p[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(h, tiny, bias));
    }
}

// Page numbers of a wave's tiles, 64 a register: those of tiles 32 g .. + 31 and of the 32
// behind.  A number outside the pool reads its last page.
struct Table {
    int32_t near, far;
    int g;
};
__device__ __forceinline__ int32_t load_pages(const int32_t* row, int n, uint32_t cap, int g, int lane) {
    return (int32_t)min((uint32_t)row[min(64 * g + lane, n - 1)], cap - 1);
}
__device__ __forceinline__ uint32_t page_of(const Table& p, int j) {   // j: the page's place, within the two
    const int at = j & 63;
    return (uint32_t)((j >> 6) == p.g ? __builtin_amdgcn_readlane(p.near, at) : __builtin_amdgcn_readlane(p.far, at));
}

__device__ __forceinline__ float pair_sum(float v) {   // of lane and lane ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// State of a row over a unit's pages.  K's and V's values are c times their token's scale; K's
// enter the products as k_i = 2^-24 (2 c + 32), V's as c:
//   z   = kScale2 2^23 s_k (sum_i q_i k_i - 2^-19 sum_i q_i)
//   o   = sum_t P_t c_t,   P_t = fp16(2^(z_t - m + shift) s_v)
// so a record of K is decoded by bit operations alone; the correction of z starts the product's
// accumulator.  ROUND: K's values are rounded to fp16 as the cache's readers see them, for weights
// that agree with a dense attention's in 32 bits: c's own pairs, times the scale.
struct PageState {
    float m, l;                                // reference, sum of 2^(z - m + shift)
    float shift;                               // kPShift less the exponent of V's largest scale so far: P's range is that of a scale of 1
    float limit;                               // a logarithm of a weight beyond it raises the reference
    f4_t o[8];
};
constexpr float kUnit = 8388608.0f;            // 2^23
__device__ __forceinline__ void rescale(PageState& st, float f) {
    st.l *= f;
#pragma unroll
    for (int mm = 0; mm < 8; mm++)
#pragma unroll
        for (int i = 0; i < 4; i++) st.o[mm][i] *= f;
}
template <int CTRL>
__device__ __forceinline__ float dppf(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// sum and maximum over the lanes that hold a row
__device__ __forceinline__ float quarters_sum(float v) {
    v = pair_sum(v);
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int NR>
__device__ __forceinline__ float shares_sum(float v) {   // within a quarter
    if (NR <= 8) v += dppf<0x128>(v);          // row_ror:8
    if (NR <= 4) v += dppf<0x124>(v);          // row_ror:4
    return v;
}
template <int NR>
__device__ __forceinline__ float row_max(float v) {
    if (NR <= 8) v = fmaxf(v, dppf<0x128>(v));
    if (NR <= 4) v = fmaxf(v, dppf<0x124>(v));
    return quarters_max(v);
}
// the largest of the lane's scales, and the least e with 2^e >= every one of the wave's (fp16's: -24 at least)
template <int NR>
__device__ __forceinline__ float lane_scale(const uint32_t s[4]) {
    h2_t m = __builtin_bit_cast(h2_t, s[0]);
#pragma unroll
    for (int i = 1; i < kPairs<NR>; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(h2_t, s[i]));
    return fmaxf((float)m[0], (float)m[1]);
}
template <int NR>
__device__ __forceinline__ float scale_log(const uint32_t s[4]) {
    const float m = row_max<NR>(lane_scale<NR>(s));   // the lanes of a quarter have the same tokens
    return fmaxf((float)((int)((__float_as_uint(m) + 0x7fffffu) >> 23) - 127), -24.f);
}

// One tile: scores s[y][i] of token 8 (lane / 16) + 2 i + y (without their scales, or with
// them where ROUND), V's coordinates.  With SUMS the logarithm (base 2) of the sum of the lane's page
// (lanes 0..31 hold the first page's tokens, 32..63 the second's).
template <bool SUMS, bool ROUND, int NR>
__device__ __forceinline__ float attend(const f4_t s[2], const uint32_t ks[4], const uint32_t vs[4], uint32_t word,
                                        const u32x4_t vq[8], int lane, PageState& st) {
    constexpr int N = 2 * kPairs<NR>;          // tokens that the lane weighs
    float z[N];
#pragma unroll
    for (int i = 0; i < N; i++) {              // from the lane that has them, r of the quarter, a share at a time
        int x = __float_as_int(s[i & 1][i >> 1]);
#define LQ_SHARE(A) x = __builtin_amdgcn_update_dpp(x, __float_as_int(s[i & 1][(i >> 1) + (A) * kPairs<NR>]), \
                                                    0x110 + (A) * NR, 0xf, NR == 8 ? 0xc : 1 << (A), false)   // row_shr
        if constexpr (NR <= 8) LQ_SHARE(1);
        if constexpr (NR == 4) {
            LQ_SHARE(2);
            LQ_SHARE(3);
        }
#undef LQ_SHARE
        z[i] = __int_as_float(x);
    }
    float off = (st.m == -INFINITY ? 0.f : -st.m) + st.shift;
#pragma unroll
    for (int i = 0; i < N; i++)
        z[i] = ROUND ? __builtin_fmaf(z[i], kScale2, off)
                     : __builtin_fmaf((float)__builtin_bit_cast(h2_t, ks[i >> 1])[i & 1], z[i] * (kScale2 * kUnit), off);
    if (word != ~0u) {
        const uint32_t own = word >> (8 * (lane >> 4) + (lane & 15) / NR * N);
#pragma unroll
        for (int i = 0; i < N; i++) z[i] = (own >> i) & 1u ? z[i] : -INFINITY;
    }
    float mx = fmaxf(z[0], z[1]);
#pragma unroll
    for (int i = 2; i < N; i += 2) mx = fmaxf(fmaxf(mx, z[i]), z[i + 1]);
    if (__any(mx > st.limit)) {                // rare after the first tile
        const float mn = row_max<NR>(mx);      // what the reference is raised by, in the rows that pass it
        const bool up = mn > st.limit;
        const float by = up ? mn - st.shift : 0.f;
        rescale(st, st.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(-by));   // nothing has been summed without one
        if (up) st.m = (st.m == -INFINITY ? 0.f : st.m) + by;
        st.limit = st.m == -INFINITY ? -INFINITY : st.shift + kLazy;
#pragma unroll
        for (int i = 0; i < N; i++) z[i] -= by;
        off -= by;
    }
    uint32_t p[4];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const float u = __builtin_amdgcn_exp2f(z[2 * i]), v = __builtin_amdgcn_exp2f(z[2 * i + 1]);
        const h2_t sv = __builtin_bit_cast(h2_t, vs[i]);
        sum += u + v;
        p[i] = pair_h(u * (float)sv[0], v * (float)sv[1]);   // the product's operand: one rounding, 2^-11 of it at most
    }
    st.l += sum;
    // back to lane r, which has row r's eight tokens in the product (what the others have goes
    // into columns that are not read)
    if constexpr (NR == 8) {
#pragma unroll
        for (int i = 0; i < 2; i++) p[2 + i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p[i], 0x108, 0xf, 0xf, false);   // row_shl
    }
    if constexpr (NR == 4) {
        p[1] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p[0], 0x104, 0xf, 0xf, false);
        p[2] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p[0], 0x108, 0xf, 0xf, false);
        p[3] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p[0], 0x10c, 0xf, 0xf, false);
    }
    const h8_t pb = as_h8(p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int mm = 0; mm < 8; mm++)
        st.o[mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, vq[mm]), pb, st.o[mm], 0, 0, 0);
    return SUMS ? __builtin_amdgcn_logf(pair_sum(shares_sum<NR>(sum))) - off + kPShift : 0.f;
}

__device__ __forceinline__ void zero_out(const PagedArgs& A, int b, int tid, int threads) {
    const int n = A.heads * A.group * (kHd / 8);
    for (int i = tid; i < n; i += threads)
        *reinterpret_cast<uint4*>(A.out + b * A.ob + (i >> 4) * A.oh + 8 * (i & 15)) = make_uint4(0u, 0u, 0u, 0u);
}

template <bool BF16>
__device__ __forceinline__ void put8(const PagedArgs& A, uint32_t unit, int row, int d, const float x[8], float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float u = x[2 * i] * inv, v = x[2 * i + 1] * inv;
        w[i] = BF16 ? (uint32_t)f2bf(u) | ((uint32_t)f2bf(v) << 16) : pair_h(u, v);
    }
    const int b = (int)(unit >> 16), h = (int)(unit & 0xffffu);
    *reinterpret_cast<uint4*>(A.out + b * A.ob + (int64_t)(h * A.group + row) * A.oh + d) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int64_t lse_at(const PagedArgs& A, uint32_t unit, int row) {
    return ((int64_t)(unit >> 16) * A.heads + (unit & 0xffffu)) * A.group + row;
}

// The lengths of up to 64 sequences, one a lane (per == 1), or from memory.
struct Lens {
    int pages, tail;
};
__device__ __forceinline__ Len len_at(const PagedArgs& A, const Lens& mine, int b) {
    if (A.per > 1) return len_of(A, b);
    Len l;
    l.pages = __builtin_amdgcn_readlane(mine.pages, b);
    l.tail = __builtin_amdgcn_readlane(mine.tail, b);
    l.page_tiles = (l.pages + 1) >> 1;
    l.tiles = l.page_tiles + ((l.tail + 31) >> 5);
    l.places = l.tiles ? (uint32_t)(l.tiles + A.ahead) : 0u;
    return l;
}
template <bool BF16, bool SUMS, bool BIG, int NR, int W, bool WHOLE>
__global__ __launch_bounds__(W * 64, 2) void k_paged(PagedArgs A) {
    constexpr bool ROUND = SUMS;
    extern __shared__ __align__(16) char s_dyn[];
    // pieces in the order of the list: wave w's first (2 w), which ends its unit there, and its last (2 w + 1)
    __shared__ uint32_t s_unit[2 * W];
    __shared__ int s_begins[2 * W];
    __shared__ uint32_t s_end;                 // where the list's unit that is begun here and not ended ends
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4, G = A.group;
    const int slot = G * kMRow * 4;            // bytes of a piece
    const int last_area = max(kPatch, slot), stride = last_area + slot;
    char* mine = s_dyn + wave * stride;        // exceptions, then the wave's last piece; behind it its first
    u32x4_t* area = reinterpret_cast<u32x4_t*>(mine);

    if (tid < 2 * W) s_unit[tid] = ~0u;
    // ---- the workgroup's share of the list, found by every wave for itself
    uint32_t lo, hi, share = 0, longer = 0;    // the first `longer` workgroups have one place more
    Lens lens = {0, 0};
    uint32_t own = 0, before = 0;
    int b = 0, h = 0;
    Len L;
    const uint32_t me = blockIdx.x;
    if (WHOLE) {
        b = blockIdx.y;
        h = blockIdx.x;
        L = len_of(A, b);
        lo = 0;
        hi = L.places;
        if (hi == 0 && h == 0) zero_out(A, b, tid, W * 64);
    } else {
        for (int i = lane * A.per; i < min((lane + 1) * A.per, A.n_seq); i++) {
            const Len l = len_of(A, i);
            lens = {l.pages, l.tail};
            own += l.places * A.heads;
        }
        // the sums up to each lane: of the lanes of a row, then of the rows
        uint32_t upto = own;
#define LQ_UPTO(CTRL, ROWS) upto += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, CTRL, ROWS, 0xf, false)
        LQ_UPTO(0x111, 0xf);                   // row_shr:1, 2, 4, 8
        LQ_UPTO(0x112, 0xf);
        LQ_UPTO(0x114, 0xf);
        LQ_UPTO(0x118, 0xf);
        LQ_UPTO(0x142, 0xa);                   // row_bcast:15 to the second and fourth
        LQ_UPTO(0x143, 0xc);                   // row_bcast:31 to the last two
#undef LQ_UPTO
        const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        before = upto - own;
        for (int i = blockIdx.x; i < A.n_seq; i += gridDim.x)
            if (len_at(A, lens, i).tiles == 0) zero_out(A, i, tid, W * 64);
        const uint32_t groups = max(1u, min((uint32_t)gridDim.x, (total + W - 1) / W));
        if (me >= groups) {
            if (tid == 0) A.desc[me] = {~0u, 0};
            return;
        }
        share = total / groups;
        longer = total % groups;
        lo = me * share + min(me, longer);
        hi = lo + share + (me < longer ? 1u : 0u);
    }
    __syncthreads();
    const uint32_t part = (hi - lo) / W, rest = (hi - lo) % W;
    uint32_t pos = lo + wave * part + min((uint32_t)wave, rest);
    const uint32_t end = pos + part + ((uint32_t)wave < rest ? 1u : 0u);

    if (pos < end) {
        uint32_t place = pos;                  // within the unit
        if (!WHOLE) {
            const uint64_t there = __ballot(pos >= before && pos - before < own);
            const int from = __ffsll((long long)there) - 1;
            uint32_t rem = pos - (uint32_t)__builtin_amdgcn_readlane((int)before, from);
            b = from * A.per;
            L = len_at(A, lens, b);
            for (int k = 1; k < A.per; k++) {
                const uint32_t n = L.places * A.heads;
                if (rem < n || b + 1 >= A.n_seq) break;
                rem -= n;
                L = len_of(A, ++b);
            }
            const uint32_t places = max(L.places, 1u);
            h = (int)(rem / places);
            place = rem % places;
        }
        for (;;) {
            const uint32_t unit = unit_of(b, h);
            const uint32_t take = min(L.places - place, end - pos);
            const int t = max((int)place - A.ahead, 0), n = max((int)(place + take) - A.ahead, 0) - t;
            if (n == 0) break;                 // the share ends before the unit's tiles
            h8_t q[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (col < G) w = load_row8<BF16>(A.q.p + b * A.q.sb + (int64_t)(h * G + col) * A.q.sh + 32 * c + 8 * g);
                q[c] = __builtin_bit_cast(h8_t, w);
            }
            FewState st;
            st.m = -INFINITY;
            st.l = 0.f;
            float l32 = 0.f;                   // the sum in 32 bits throughout
#pragma unroll
            for (int mm = 0; mm < 8; mm++) st.o[mm] = f4_t{0.f, 0.f, 0.f, 0.f};

            // ---- the pages' tiles
            const int pe = min(t + n, L.page_tiles);
            if (t < pe) {
                const int32_t* row = A.pages + b * A.width;
                const uint32_t cap = (uint32_t)A.k.r.cap_blocks, hb = (uint32_t)h * cap;
                Table pg;
                pg.g = t >> 5;
                pg.near = load_pages(row, L.pages, cap, pg.g, lane);
                pg.far = load_pages(row, L.pages, cap, pg.g + 1, lane);
                f4_t s0 = {0.f, 0.f, 0.f, 0.f};
                if (!ROUND) {                  // -2^-19 sum_i q_i
                    float x = 0.f;
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int i = 0; i < 8; i++) x += (float)q[c][i];
                    x = quarters_sum(x) * (-0x1p-19f);
                    s0 = f4_t{x, x, x, x};
                }
                PageState ps;
                ps.m = -INFINITY;
                ps.l = 0.f;
                ps.shift = kPShift;
                ps.limit = -INFINITY;
                float largest = 0.f;           // no scale has been above it
#pragma unroll
                for (int mm = 0; mm < 8; mm++) ps.o[mm] = f4_t{0.f, 0.f, 0.f, 0.f};
                Recs rd;
                Meta2 mk, mv, nk, nv;
                Entry ek, ev;
                uint32_t x1, y1;               // blocks of the next tile; past the end the last again
                const auto blocks = [&](int tile) __attribute__((always_inline)) {
                    const int j = 2 * min(tile, pe - 1);
                    x1 = hb + page_of(pg, j);
                    y1 = hb + page_of(pg, min(j + 1, L.pages - 1));
                };
                blocks(t);
                mk = load_meta<BIG>(A.k, x1, y1, lane);
                mv = load_meta<BIG>(A.v, x1, y1, lane);
                load_k<BIG, ROUND, NR>(A, x1, y1, lane, rd);
                load_v<BIG, NR>(A, x1, y1, lane, rd);
                blocks(t + 1);
                nk = load_meta<BIG>(A.k, x1, y1, lane);
                nv = load_meta<BIG>(A.v, x1, y1, lane);
                ek = load_entry<BIG>(A.k, mk, lane & 31);
                ev = load_entry<BIG>(A.v, mv, lane & 31);
                for (int tile = t; tile < pe; tile++) {
                    const uint32_t word = 2 * tile + 1 < L.pages ? ~0u : 0xffffu;
                    f4_t s[2] = {s0, s0};
                    uint32_t p[8][4];
                    u32x4_t vq[8];             // of V: vector lane % 16's dimension, four pairs of tokens
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t ra = j & 1 ? rd.ka[j >> 1].y : rd.ka[j >> 1].x, rb = rd.kb[j >> 1];
                        if constexpr (ROUND) {
                            rec_pairs(ra, (rb >> (8 * (j & 1))) & 0xffu, p[j]);
#pragma unroll
                            for (int i = 0; i < 4; i++) p[j][i] = unbias(p[j][i]);
                        } else if (j & 1) {
                            raw_pairs<8>(ra, rb, p[j]);
                        } else {
                            raw_pairs<0>(ra, rb, p[j]);
                        }
                    }
                    if (const uint32_t most = most_of(mk)) {
                        // through 8 KB of LDS of the wave's own, the lanes with entries write over their records
#pragma unroll
                        for (int j = 0; j < 8; j++) area[64 * j + lane] = u32x4_t{p[j][0], p[j][1], p[j][2], p[j][3]};
                        wave_lds_sync();
                        each_entry<BIG>(A.k, mk, ek, most, lane, [&](uint32_t rec, const uint4& w) __attribute__((always_inline)) {
                            uint32_t e[4];
                            if constexpr (ROUND) exc_pairs(w, e);
                            else raw_entry(w, e);
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
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if constexpr (ROUND) mul_pairs<4>(p[j], __builtin_amdgcn_perm(0u, rd.kp, j & 1 ? 0x03020302u : 0x01000100u));
                        s[j & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(p[j][0], p[j][1], p[j][2], p[j][3]), q[j >> 1],
                                                                          s[j & 1], 0, 0, 0);
                    }
                    // The next tile's records, as soon as these are used (every use scheduled before the
                    // reload), and the bases of the one behind; past the end the last tile's again.
                    uint32_t ks[4], vs[4];
                    if (!ROUND) {
#pragma unroll
                        for (int i = 0; i < kPairs<NR>; i++) ks[i] = copied(rd.ks[i]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    ek = load_entry<BIG>(A.k, nk, lane & 31);
                    mk = {copied(nk.base), copied(nk.count)};
                    load_k<BIG, ROUND, NR>(A, x1, y1, lane, rd);
                    {
                        const uint32_t aw[8] = {rd.va[0].x, rd.va[0].y, rd.va[0].z, rd.va[0].w,
                                                rd.va[1].x, rd.va[1].y, rd.va[1].z, rd.va[1].w};
                        pairs_tok<0, 0>(aw[0], aw[1], rd.vb.x, vq);
                        pairs_tok<16, 1>(aw[2], aw[3], rd.vb.x, vq);
                        pairs_tok<0, 2>(aw[4], aw[5], rd.vb.y, vq);
                        pairs_tok<16, 3>(aw[6], aw[7], rd.vb.y, vq);
                    }
                    if (const uint32_t most = most_of(mv)) {
#pragma unroll
                        for (int j = 0; j < 8; j++) area[64 * j + lane] = vq[j];
                        wave_lds_sync();
                        each_entry<BIG>(A.v, mv, ev, most, lane, [&](uint32_t rec, const uint4& v) __attribute__((always_inline)) {
                            uint32_t e[4];
                            exc_pairs(v, e);
                            const uint32_t tok = 16 * (lane >> 5) + (rec & 15);
                            uint16_t* w = reinterpret_cast<uint16_t*>(area + 16 * (tok >> 3) + (rec >> 4)) + (tok & 7);
#pragma unroll
                            for (int i = 0; i < 8; i++) w[512 * i] = (uint16_t)(i & 1 ? e[i >> 1] >> 16 : e[i >> 1]);
                        });
                        wave_lds_sync();
#pragma unroll
                        for (int j = 0; j < 8; j++) vq[j] = area[64 * j + lane];
                        wave_lds_sync();
                    }
                    if (__any(lane_scale<NR>(rd.vs) > largest)) {
                        const float e = scale_log<NR>(rd.vs), by = kPShift - e - ps.shift;
                        rescale(ps, __builtin_amdgcn_exp2f(by));
                        ps.shift += by;
                        ps.limit += by;
                        largest = __builtin_amdgcn_exp2f(e);
                    }
#pragma unroll
                    for (int i = 0; i < kPairs<NR>; i++) vs[i] = copied(rd.vs[i]);
                    __builtin_amdgcn_sched_barrier(0);
                    ev = load_entry<BIG>(A.v, nv, lane & 31);
                    mv = {copied(nv.base), copied(nv.count)};
                    load_v<BIG, NR>(A, x1, y1, lane, rd);
                    if (((tile + 2) >> 5) == pg.g + 2) {
                        pg.g++;
                        pg.near = pg.far;
                        pg.far = load_pages(row, L.pages, cap, pg.g + 1, lane);
                    }
                    blocks(tile + 2);
                    nk = load_meta<BIG>(A.k, x1, y1, lane);
                    nv = load_meta<BIG>(A.v, x1, y1, lane);
                    const float z = attend<SUMS, ROUND, NR>(s, ks, vs, word, vq, lane, ps);
                    if (SUMS) {
                        const int j = 2 * tile + (lane >> 5);
                        if (!(g & 1) && col < G && j < L.pages) A.z[(((int64_t)b * A.heads + h) * A.width + j) * G + col] = z;
                    }
                }
                // on as the tail's rows are taken
                const float f = __builtin_amdgcn_exp2f(kPShift - ps.shift);
                st.m = ps.m;
                st.l = l32 = shares_sum<NR>(ps.l) * f;
#pragma unroll
                for (int mm = 0; mm < 8; mm++)
#pragma unroll
                    for (int i = 0; i < 4; i++) st.o[mm][i] = ps.o[mm][i] * f;
            }
            // ---- the tail's
            for (int tile = max(t, L.page_tiles); tile < t + n; tile++) {
                const int t0 = 32 * (tile - L.page_tiles), have = min(L.tail - t0, 32);
                const uint32_t word = have == 32 ? ~0u : (1u << have) - 1u;
                f4_t s[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
                uint32_t vp[4][8];
                uint4 w[2][4];
                const uint16_t* p = A.tk.p + b * A.tk.sb + h * A.tk.sh;
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int tok = min(8 * (col >> 2) + 2 * (col & 3) + y, have - 1);
                        w[y][c] = *reinterpret_cast<const uint4*>(p + (t0 + tok) * A.tk.st + 32 * c + 8 * g);
                    }
                __builtin_amdgcn_sched_barrier(0);
                rows_v<BF16>(A.tv.p + b * A.tv.sb + h * A.tv.sh, A.tv.st, t0, have, word, lane, vp);
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        s[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            __builtin_bit_cast(h8_t, BF16 ? bf_to_h(w[y][c]) : w[y][c]), q[c], s[y], 0, 0, 0);
                const float was = st.m;
                few_attend(s, word, word == ~0u, vp, lane, st);
                if (SUMS) {                    // few_attend's sum is of the rounded weights: these few again
                    if (was != st.m) l32 *= __builtin_amdgcn_exp2f(was - st.m);
                    const float off = (st.m == -INFINITY ? 0.f : -st.m) + kPShift;
#pragma unroll
                    for (int i = 0; i < 8; i++) l32 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[i & 1][i >> 1], kScale2, off));
                }
            }
            // ---- the unit is written out, or its piece kept
            const float l = quarters_sum(st.l);
            if (SUMS) l32 = quarters_sum(l32);
            const bool ends = t + n == L.tiles;
            if (t == 0 && ends) {
                if (col < G) {
                    const float inv = 1.f / l;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x[8] = {st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i],
                                            st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]};
                        put8<BF16>(A, unit, col, 8 * (4 * g + i), x, inv);
                    }
                    if (SUMS && g == 0) A.lse[lse_at(A, unit, col)] = st.m + __builtin_amdgcn_logf(l32);
                }
            } else {
                float* to = reinterpret_cast<float*>(mine + (ends ? last_area : 0)) + col * kMRow;
                if (!ends) wave_lds_sync();
                if (col < G) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        *reinterpret_cast<f4_t*>(to + 8 * (4 * g + i)) = f4_t{st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i]};
                        *reinterpret_cast<f4_t*>(to + 8 * (4 * g + i) + 4) = f4_t{st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]};
                    }
                    if (g == 0) {
                        to[kHd] = st.m;
                        to[kHd + 1] = l;
                        if (SUMS) to[kHd + 2] = l32;
                    }
                }
                if (lane == 0) {
                    const int i = 2 * wave + (ends ? 0 : 1);
                    s_unit[i] = unit;
                    s_begins[i] = t == 0;
                    if (!ends && pos + take == hi) s_end = pos + L.places - place;
                }
            }
            pos += take;
            if (WHOLE || pos == end) break;
            place = 0;
            if (++h == A.heads) {
                h = 0;
                do {
                    if (++b >= A.n_seq) break;
                    L = len_at(A, lens, b);
                } while (L.tiles == 0);
                if (b >= A.n_seq) break;
            }
        }
    }
    __syncthreads();

    // ---- pieces joined, unit by unit, a wave's at most: 16 lanes a row, eight dimensions a lane
    Desc left = {~0u, 0};
    const int row = tid >> 4, d = 8 * (tid & 15);
    const uint32_t units = lane < 2 * W ? s_unit[lane] : ~0u;
    const uint32_t begun = (uint32_t)__ballot(lane < 2 * W && s_begins[lane & (2 * W - 1)] != 0);
    for (uint32_t open = (uint32_t)__ballot(units != ~0u); open;) {
        const int at = __ffs((int)open) - 1;
        const uint32_t unit = (uint32_t)__builtin_amdgcn_readlane((int)units, at), its = (uint32_t)__ballot(units == unit);
        open &= ~its;
        const bool begins = (begun >> at) & 1u, ends = (its & 0x55555555u) != 0u;
        if (row < G) {
            float pm[W], pl[W], p32[W];
            f4_t u[W], v[W];
#pragma unroll
            for (int w = 0; w < W; w++) {
                pm[w] = -INFINITY;
                pl[w] = p32[w] = 0.f;
                u[w] = v[w] = f4_t{0.f, 0.f, 0.f, 0.f};
                if (!((its >> (2 * w)) & 3u)) continue;
                const float* p = reinterpret_cast<const float*>(s_dyn + w * stride + ((its >> (2 * w)) & 1u ? last_area : 0)) + row * kMRow;
                pm[w] = p[kHd];
                pl[w] = p[kHd + 1];
                if (SUMS) p32[w] = p[kHd + 2];
                u[w] = *reinterpret_cast<const f4_t*>(p + d);
                v[w] = *reinterpret_cast<const f4_t*>(p + d + 4);
            }
            float m = -INFINITY, l = 0.f, l32 = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; w++) m = fmaxf(m, pm[w]);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = pm[w] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(pm[w] - m);
                l = __builtin_fmaf(pl[w], f, l);
                if (SUMS) l32 = __builtin_fmaf(p32[w], f, l32);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[e] = __builtin_fmaf(u[w][e], f, x[e]);
                    x[4 + e] = __builtin_fmaf(v[w][e], f, x[4 + e]);
                }
            }
            if (begins && ends) {
                put8<BF16>(A, unit, row, d, x, 1.f / l);
                if (SUMS && d == 0) A.lse[lse_at(A, unit, row)] = m + __builtin_amdgcn_logf(l32);
            } else {
                float* rec = A.rec + ((int64_t)(2 * me + (begins ? 1 : 0)) * G + row) * kRecF;
                *reinterpret_cast<f4_t*>(rec + 4 + d) = f4_t{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<f4_t*>(rec + 8 + d) = f4_t{x[4], x[5], x[6], x[7]};
                if (d == 0) *reinterpret_cast<f4_t*>(rec) = f4_t{m, l, l32, 0.f};
            }
        }
        if (begins && !ends) {                 // the workgroup that has the unit's last place
            const uint32_t last = s_end - 1, split = longer * (share + 1);
            left = {unit, (int32_t)((last < split ? last / (share + 1) : longer + (last - split) / share) - me)};
        }
    }
    if (tid == 0 && !WHOLE) A.desc[me] = left;
}

// The records of a unit that several workgroups share, a workgroup per row: thread
// (sub, dq) sums dimensions 4 dq .. + 3 of records sub, sub + 8, .., then the eight sums
// are joined in order.  Most workgroups find no unit: within 64 registers all are resident
// at once (2048 in two rounds, seven a compute unit: 8.0 us for 6.3).
template <bool BF16, bool SUMS>
__global__ __launch_bounds__(256, 8) void k_paged_join(PagedArgs A) {
    constexpr int kUp = 4;                     // records in flight per thread
    __shared__ __align__(16) f4_t s_o[8][32];
    __shared__ float s_m[8], s_l[8], s_l32[8];
    const int dq = threadIdx.x & 31, sub = threadIdx.x >> 5, row = blockIdx.y, wg = blockIdx.x;
    const Desc D = A.desc[wg];
    if (D.unit == ~0u) return;
    const int n = 1 + D.more;
    float m = -INFINITY, l = 0.f, l32 = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = sub; p0 < n; p0 += 8 * kUp) {
        f4_t ml[kUp];
        f4_t v[kUp];
#pragma unroll
        for (int k = 0; k < kUp; k++) {
            const int p = min(p0 + 8 * k, n - 1);
            const float* x = A.rec + ((int64_t)(2 * (wg + p) + (p ? 0 : 1)) * A.group + row) * kRecF;
            ml[k] = *reinterpret_cast<const f4_t*>(x);
            v[k] = *reinterpret_cast<const f4_t*>(x + 4 + 4 * dq);
        }
        float M = m;
#pragma unroll
        for (int k = 0; k < kUp; k++) M = p0 + 8 * k < n ? fmaxf(M, ml[k][0]) : M;
        const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M);
        o *= f0;
        l *= f0;
        l32 *= f0;
#pragma unroll
        for (int k = 0; k < kUp; k++) {
            if (p0 + 8 * k >= n) continue;
            const float f = ml[k][0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[k][0] - M);
            l = __builtin_fmaf(ml[k][1], f, l);
            if (SUMS) l32 = __builtin_fmaf(ml[k][2], f, l32);
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(v[k][c], f, o[c]);
        }
        m = M;
    }
    s_o[sub][dq] = o;
    if (dq == 0) {
        s_m[sub] = m;
        s_l[sub] = l;
        s_l32[sub] = l32;
    }
    __syncthreads();
    if (threadIdx.x >= 16) return;
    const int lane = threadIdx.x;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; k++) M = fmaxf(M, s_m[k]);
    float L = 0.f, L32 = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int k = 0; k < 8; k++) {
        const float f = s_m[k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[k] - M);
        const f4_t u = s_o[k][2 * lane], v = s_o[k][2 * lane + 1];
        L = __builtin_fmaf(s_l[k], f, L);
        if (SUMS) L32 = __builtin_fmaf(s_l32[k], f, L32);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            x[c] = __builtin_fmaf(u[c], f, x[c]);
            x[4 + c] = __builtin_fmaf(v[c], f, x[4 + c]);
        }
    }
    put8<BF16>(A, D.unit, row, 8 * lane, x, 1.f / L);
    if (SUMS && lane == 0) A.lse[lse_at(A, D.unit, row)] = M + __builtin_amdgcn_logf(L32);
}

// weights[b][j] = decay * weights[b][j] + the page's weight of this step (decay 0: that
// alone), a lane a page, the heads dealt to four waves whose sums are joined in order.  Bound
// by the latency of a wave's loads: 64 sequences of up to 512 pages, 8 heads, 4 rows 4.9 us (a
// wave for all heads 8.0).
template <int G4>   // whole rows of four, or 0 for any group
__global__ __launch_bounds__(256) void k_page_weights(PagedArgs A, float* __restrict__ w, float decay) {
    __shared__ float s_sum[4][64];
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.x * 64 + lane;
    const int n = min(max(A.n_pages[b], 0), (int)A.width);
    if ((int)blockIdx.x * 64 >= n) return;
    float sum = 0.f;
    if (j < n) {
        for (int h = wave; h < A.heads; h += 4) {
            const int64_t unit = (int64_t)b * A.heads + h;
            const float* z = A.z + (unit * A.width + j) * A.group;
            const float* lse = A.lse + unit * A.group;
            if constexpr (G4) {
#pragma unroll
                for (int r = 0; r < 4 * G4; r += 4) {
                    const f4_t x = *reinterpret_cast<const f4_t*>(z + r);
#pragma unroll
                    for (int i = 0; i < 4; i++) sum += __builtin_amdgcn_exp2f(x[i] - lse[r + i]);
                }
            } else {
                for (int r = 0; r < A.group; r++) sum += __builtin_amdgcn_exp2f(z[r] - lse[r]);
            }
        }
    }
    s_sum[wave][lane] = sum;
    __syncthreads();
    if (wave || j >= n) return;
    sum = (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]);
    float* to = w + b * A.width + j;
    *to = decay == 0.f ? sum : __builtin_fmaf(decay, *to, sum);
}

// ---------------------------------------------------------------- eviction --

struct EvictArgs {
    const int32_t* pages;
    const int32_t* n_pages;
    const float* weights;
    int64_t width;
    int keep, sink, recent;
    int32_t* out_pages;
    int32_t* out_n;
    float* out_weights;
    int32_t* freed;
};

// larger weights first, NaN above all, -0 as 0
__device__ __forceinline__ uint32_t weight_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64, kBins = 2048;

// The room-th largest weight of a sequence's pages that may go, by a radix search of 11, 11
// and 10 bits (that ends where all of a bin stay), then one pass in the order of the pages,
// each wave a part of them.  A sequence of up to 8192 pages is a workgroup's, N of them a
// lane in registers, read once.  Longer ones (N = 0) are searched by `parts` workgroups each
// of which looks at all of it and writes its part: the search is repeated on compute units
// that would idle (4 sequences of 65536 pages: 46 us, one workgroup each 80).  1 / 64 / 256
// tables of 8192 pages 13.8 / 17.0 / 19.5 us (N = 0: 15.7 / 16.9 / 20.4), of 16384 with 16 a
// lane 21.2 / 26.0 / 29.6 (20.9 / 23.0 / 31.0).  Bound by latency with few pages (1024: 5.4 us),
// by instructions with many.
template <int N>
__global__ __launch_bounds__(kEvictThreads) void k_evict(EvictArgs A, int parts) {
    __shared__ uint32_t s_bin[kBins];
    __shared__ uint32_t s_part[kEvictWaves], s_tie[2][kEvictWaves], s_sure[2][kEvictWaves];
    __shared__ uint32_t s_pick, s_left, s_in;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = N ? blockIdx.x : blockIdx.x / parts, part = N ? 0 : blockIdx.x % parts;
    const float* weights = A.weights + b * A.width;
    const int32_t* pages = A.pages + b * A.width;
    const int n = min(max(A.n_pages[b], 0), (int)A.width);
    const int lo = min(A.sink, n), hi = max(lo, n - A.recent);
    const bool all = n <= A.keep;
    uint32_t room = all ? 0u : (uint32_t)max(0, A.keep - lo - (n - hi));
    const uint32_t kept_n = all ? (uint32_t)n : (uint32_t)lo + (uint32_t)(n - hi) + room;
    const bool some = room > 0;
    // steps of 64 pages: those before the workgroup's part, and the wave's of the part
    const int tiles = (n + 63) / 64, t0 = N ? 0 : (int)((int64_t)tiles * part / parts), t1 = N ? tiles : (int)((int64_t)tiles * (part + 1) / parts);
    const int per = (t1 - t0 + kEvictWaves - 1) / kEvictWaves, mine = t0 + wave * per, steps = max(0, min(per, t1 - mine));
    constexpr int C = N > 0 && N < 8 ? N : 8;  // steps whose loads go out together
    constexpr int R = N ? N : 1;
    float w[R];
    auto weight = [&](int t) __attribute__((always_inline)) { return weights[min(64 * t + lane, n - 1)]; };
    if (N) {
#pragma unroll
        for (int i = 0; i < R; i++) w[i] = i < steps ? weight(mine + i) : 0.f;
    }
    // f(page's place, weight, open: may go, in: there is such a page, its number where PAGES)
    // for `count` steps from `first` on, `stride` apart
    auto chunk = [&](auto numbers, int t, int stride, int count, const float* x, auto f) __attribute__((always_inline)) {
        int32_t page[C];
#pragma unroll
        for (int i = 0; i < C; i++)
            page[i] = decltype(numbers)::value && i < count ? pages[min(64 * (t + i * stride) + lane, n - 1)] : 0;
#pragma unroll
        for (int i = 0; i < C; i++) {
            if (i >= count) break;
            const int j = 64 * (t + i * stride) + lane;
            f(j, x[i], j >= lo && j < hi, j < n, page[i]);
        }
    };
    auto from_memory = [&](auto numbers, int first, int stride, int count, auto f) __attribute__((always_inline)) {
        float x[C];
        int i0 = 0;
        for (; i0 + C <= count; i0 += C) {
#pragma unroll
            for (int i = 0; i < C; i++) x[i] = weight(first + (i0 + i) * stride);
            chunk(numbers, first + i0 * stride, stride, C, x, f);
        }
        if (i0 < count) {
#pragma unroll
            for (int i = 0; i < C; i++) x[i] = weight(min(first + (i0 + i) * stride, tiles - 1));
            chunk(numbers, first + i0 * stride, stride, count - i0, x, f);
        }
    };
    auto each = [&](auto numbers, auto f) __attribute__((always_inline)) {   // of the wave's part
        if constexpr (N > 0) {
#pragma unroll
            for (int i = 0; i < N; i += C)
                if (i < steps) chunk(numbers, mine + i, 1, steps - i, w + i, f);
        } else {
            from_memory(numbers, mine, 1, steps, f);
        }
    };
    const std::false_type no;
    const std::true_type yes;
    uint32_t prefix = 0;                       // the bits found so far, those from `shift` on
    int shift = 32;
    if (some) {
        for (int digit = 0; digit < 3; digit++) {
            const int bits = digit == 2 ? 10 : 11, up = shift;
            shift -= bits;
            for (int i = tid; i < kBins; i += kEvictThreads) s_bin[i] = 0u;
            __syncthreads();
            auto count = [&](int, float x, bool open, bool, int32_t) __attribute__((always_inline)) {
                const uint32_t k = weight_key(x);
                if (open && (digit == 0 || k >> up == prefix)) atomicAdd(&s_bin[(k >> shift) & ((1u << bits) - 1u)], 1u);
            };
            if constexpr (N > 0) each(no, count);
            else from_memory(no, wave, kEvictWaves, (tiles - wave + kEvictWaves - 1) / kEvictWaves, count);
            __syncthreads();
            // bins from the largest down, two a thread
            const uint32_t c0 = s_bin[kBins - 1 - 2 * tid], c1 = s_bin[kBins - 2 - 2 * tid];
            uint32_t upto = c0 + c1;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t x = __shfl_up(upto, o, 64);
                upto += lane >= o ? x : 0u;
            }
            if (lane == 63) s_part[wave] = upto;
            __syncthreads();
            for (int v = 0; v < wave; v++) upto += s_part[v];
            const uint32_t before = upto - c0 - c1;
            if (before < room && room <= upto) {
                const bool second = room > before + c0;
                s_pick = (uint32_t)(kBins - 1 - 2 * tid - (second ? 1 : 0));
                s_left = room - before - (second ? c0 : 0u);
                s_in = second ? c1 : c0;
            }
            __syncthreads();
            prefix = prefix << bits | s_pick;
            room = s_left;
            if (room == s_in) break;           // the same in all threads
            __syncthreads();
        }
    }
    if (!some) shift = 0;
    // kept: the protected, what is above the bits, and the first `room` of those that have them
    uint32_t ties = 0, sure = 0;
    auto tally = [&](int, float x, bool open, bool in, int32_t) __attribute__((always_inline)) {
        const uint32_t k = weight_key(x) >> shift;
        ties += __builtin_popcountll(__ballot(open && some && k == prefix));
        sure += __builtin_popcountll(__ballot(in && (all || !open || (some && k > prefix))));
    };
    if (!N && t0 > 0) from_memory(no, wave, kEvictWaves, max(0, (t0 - wave + kEvictWaves - 1) / kEvictWaves), tally);
    if (lane == 0) {
        s_tie[0][wave] = ties;
        s_sure[0][wave] = sure;
    }
    ties = sure = 0;
    each(no, tally);
    if (lane == 0) {
        s_tie[1][wave] = ties;
        s_sure[1][wave] = sure;
    }
    __syncthreads();
    uint32_t tie = 0, to = 0;                  // of those with the bits, and of all kept, before the wave's part
#pragma unroll
    for (int v = 0; v < kEvictWaves; v++) {
        tie += s_tie[0][v];
        to += s_sure[0][v];
    }
    to += min(tie, room);
    for (int v = 0; v < wave; v++) {
        to += s_sure[1][v] + min(s_tie[1][v], tie < room ? room - tie : 0u);
        tie += s_tie[1][v];
    }
    int32_t* out_pages = A.out_pages + b * A.width;
    float* out_weights = A.out_weights + b * A.width;
    int32_t* freed = A.freed + b * A.width;
    const uint64_t below = (1ull << lane) - 1ull;
    each(yes, [&](int j, float x, bool open, bool in, int32_t page) __attribute__((always_inline)) {
        const uint32_t k = weight_key(x) >> shift;
        const uint64_t eq = __ballot(open && some && k == prefix);
        const bool keep = in && (all || !open || (some && (k > prefix || (k == prefix && tie + __builtin_popcountll(eq & below) < room))));
        const uint64_t kept = __ballot(keep);
        const uint32_t p = to + __builtin_popcountll(kept & below);
        if (keep) {
            out_pages[p] = page;
            out_weights[p] = x;
        } else if (in) {
            freed[(uint32_t)j - p] = page;
        }
        tie += __builtin_popcountll(eq);
        to += __builtin_popcountll(kept);
    });
    for (int64_t j = (int64_t)kept_n + part * kEvictThreads + tid; j < A.width; j += (int64_t)kEvictThreads * parts) {
        out_pages[j] = -1;
        out_weights[j] = 0.f;
    }
    for (int64_t j = (int64_t)(n - kept_n) + part * kEvictThreads + tid; j < A.width; j += (int64_t)kEvictThreads * parts) freed[j] = -1;
    if (tid == 0 && part == 0) A.out_n[b] = (int32_t)kept_n;
}

// ------------------------------------------------------------------- plan --

struct Plan {
    int grid;
    bool whole;                                // a workgroup a unit, instead of equal shares
    int64_t rec, desc, lse, z, bytes;          // bytes before each, and in all
};
bool plan(int64_t n_seq, int64_t heads, int64_t group, int64_t width, int64_t tail_cap, bool weights, Plan* p) {
    if (n_seq < 1 || heads < 1 || group < 1 || group > 16 || width < 0 || tail_cap < 0 || width > INT_MAX / 64 ||
        tail_cap > INT_MAX / 64 || n_seq > 65535 || heads > 65535 || n_seq * heads > INT_MAX / 16)
        return false;
    const int64_t tiles = (width + 1) / 2 + (tail_cap + 31) / 32;
    if (tiles + kAhead > INT_MAX / (n_seq * heads)) return false;
    // (no tile at all: the sequences' zeros are dealt to the workgroups)
    const int64_t most = tiles ? (n_seq * heads * tiles + kWaves - 1) / kWaves : n_seq;
    p->whole = tiles <= kWhole && n_seq * heads <= kGroups;
    p->grid = (int)(p->whole ? n_seq * heads : most < kGroups ? most : kGroups);
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    p->rec = 0;
    p->desc = p->rec + (p->whole ? 256 : up(2 * p->grid * group * kRecF * 4));
    p->lse = p->desc + up(p->whole ? 0 : p->grid * (int64_t)sizeof(Desc));
    p->z = p->lse + (weights ? up(n_seq * heads * group * 4) : 0);
    p->bytes = p->z + (weights ? up(n_seq * heads * group * width * 4) : 0);
    return true;
}

bool pool_ok(const lq_pages* p) {
    const lq_resident* r = p ? &p->r : nullptr;
    return r && r->a && r->b && r->mask && r->meta && r->scale && r->n_heads > 0 && r->cap_blocks > 0 && r->exc_cap >= 0 &&
           r->exc_cap <= INT_MAX && r->cap_blocks <= INT_MAX / r->n_heads && (r->exc_cap == 0 || (r->exc && p->rec));
}
bool rows_ok(const lq_rows* r) {
    return r && r->p && ((uintptr_t)r->p & 15) == 0 && r->stride_b % 8 == 0 && r->stride_h % 8 == 0 && r->stride_t % 8 == 0;
}
Rows rows_of(const lq_rows* r) { return {static_cast<const uint16_t*>(r->p), r->stride_b, r->stride_h, r->stride_t}; }

template <bool BF16, bool SUMS, bool BIG, int W, bool WHOLE>
void paged_launch(const PagedArgs& A, const dim3& g, hipStream_t s) {
    const int slot = A.group * kMRow * 4;
    const size_t lds = (size_t)W * ((slot > kPatch ? slot : kPatch) + slot);
    const dim3 wg(W * 64);
    if (A.group <= 4) hipLaunchKernelGGL((k_paged<BF16, SUMS, BIG, 4, W, WHOLE>), g, wg, lds, s, A);
    else if (A.group <= 8) hipLaunchKernelGGL((k_paged<BF16, SUMS, BIG, 8, W, WHOLE>), g, wg, lds, s, A);
    else hipLaunchKernelGGL((k_paged<BF16, SUMS, BIG, 16, W, WHOLE>), g, wg, lds, s, A);
}
template <bool BF16, bool SUMS, bool BIG>
void paged_launch(const PagedArgs& A, bool whole, int grid, hipStream_t s) {
    if (whole) {
        const dim3 g((unsigned)A.heads, (unsigned)A.n_seq);
        if (grid <= kGroups / 2) paged_launch<BF16, SUMS, BIG, kWholeWaves, true>(A, g, s);
        else paged_launch<BF16, SUMS, BIG, kWaves, true>(A, g, s);
        return;
    }
    paged_launch<BF16, SUMS, BIG, kWaves, false>(A, dim3((unsigned)grid), s);
    hipLaunchKernelGGL((k_paged_join<BF16, SUMS>), dim3((unsigned)grid, (unsigned)A.group), dim3(256), 0, s, A);
}
template <bool BF16, bool SUMS>
void paged_launch(const PagedArgs& A, const Plan& p, bool big, hipStream_t s) {
    if (big) paged_launch<BF16, SUMS, true>(A, p.whole, p.grid, s);
    else paged_launch<BF16, SUMS, false>(A, p.whole, p.grid, s);
}

}  // namespace

extern "C" {

int64_t lq_paged_attn_workspace(int64_t n_seq, int64_t heads, int group, int64_t max_pages, int64_t tail_cap, int weights) {
    Plan p;
    return plan(n_seq, heads, group, max_pages, tail_cap, weights != 0, &p) ? p.bytes : -1;
}

int lq_paged_attention(const lq_pages *k, const lq_pages *v, const lq_rows *q, int64_t n_seq, int group,
                       const int32_t *d_pages, int64_t max_pages, const int32_t *d_n_pages, const lq_rows *tail_k,
                       const lq_rows *tail_v, int64_t tail_cap, const int32_t *d_tail_len, float *d_weights, float decay,
                       int dtype, void *d_work, int64_t work_bytes, const lq_rows *out, hipStream_t s) {
    if (!pool_ok(k) || !pool_ok(v) || k->r.n_heads != v->r.n_heads || k->r.cap_blocks != v->r.cap_blocks || !rows_ok(q) ||
        !rows_ok(out) || !d_n_pages || (max_pages > 0 && !d_pages) || !d_work || ((uintptr_t)d_work & 15) ||
        (dtype != LQ_F16 && dtype != LQ_BF16))
        return LQ_ERR_ARG;
    if (tail_cap > 0 && (!rows_ok(tail_k) || !rows_ok(tail_v))) return LQ_ERR_ARG;
    Plan p;
    if (!plan(n_seq, k->r.n_heads, group, max_pages, tail_cap, d_weights != nullptr, &p) || work_bytes < p.bytes)
        return LQ_ERR_ARG;
    PagedArgs A{};
    A.k = *k;
    A.v = *v;
    // an empty exception list is read at its first entry and the value not used
    for (lq_pages* p : {&A.k, &A.v}) {
        if (p->r.exc_cap) continue;
        p->r.exc = reinterpret_cast<int16_t*>(p->r.a);
        p->rec = p->r.b;
    }
    A.pages = d_pages;
    A.n_pages = d_n_pages;
    A.tail_len = d_tail_len;
    A.width = max_pages;
    A.tail_cap = tail_cap;
    A.q = rows_of(q);
    if (tail_cap > 0) { A.tk = rows_of(tail_k); A.tv = rows_of(tail_v); }
    A.out = static_cast<uint16_t*>(out->p);
    A.ob = out->stride_b;
    A.oh = out->stride_h;
    A.n_seq = (int)n_seq;
    A.heads = (int)k->r.n_heads;
    A.group = group;
    A.per = (int)((n_seq + 63) / 64);
    A.ahead = p.whole ? 0 : kAhead;
    char* w = static_cast<char*>(d_work);
    A.rec = reinterpret_cast<float*>(w + p.rec);
    A.desc = reinterpret_cast<Desc*>(w + p.desc);
    A.lse = reinterpret_cast<float*>(w + p.lse);
    A.z = reinterpret_cast<float*>(w + p.z);
    const bool big = k->r.n_heads * k->r.cap_blocks > (int64_t)(UINT32_MAX / 1024) ||
                     (k->r.exc_cap > v->r.exc_cap ? k->r.exc_cap : v->r.exc_cap) > (int64_t)(UINT32_MAX / 16);
    if (dtype == LQ_BF16) {
        if (d_weights) paged_launch<true, true>(A, p, big, s);
        else paged_launch<true, false>(A, p, big, s);
    } else {
        if (d_weights) paged_launch<false, true>(A, p, big, s);
        else paged_launch<false, false>(A, p, big, s);
    }
    if (d_weights && max_pages > 0) {
        const dim3 wg((unsigned)((max_pages + 63) / 64), (unsigned)n_seq);
        if (group == 4) hipLaunchKernelGGL(k_page_weights<1>, wg, dim3(256), 0, s, A, d_weights, decay);
        else if (group == 8) hipLaunchKernelGGL(k_page_weights<2>, wg, dim3(256), 0, s, A, d_weights, decay);
        else hipLaunchKernelGGL(k_page_weights<0>, wg, dim3(256), 0, s, A, d_weights, decay);
    }
    return launch_status();
}

int lq_evict_pages(const int32_t *d_pages, const int32_t *d_n_pages, const float *d_weights, int64_t n_seq,
                   int64_t max_pages, int64_t keep, int64_t sink, int64_t recent, int32_t *d_out_pages, int32_t *d_out_n,
                   float *d_out_weights, int32_t *d_freed, hipStream_t s) {
    if (!d_pages || !d_n_pages || !d_weights || !d_out_pages || !d_out_n || !d_out_weights || !d_freed || n_seq < 1 ||
        n_seq > UINT32_MAX / kEvictThreads || max_pages < 1 || max_pages > INT_MAX / 2 || sink < 0 || recent < 0 || sink > INT_MAX / 2 ||
        recent > INT_MAX / 2 || keep < sink + recent || keep > INT_MAX)
        return LQ_ERR_ARG;
    const EvictArgs A = {d_pages, d_n_pages, d_weights, max_pages, (int)keep, (int)sink, (int)recent,
                         d_out_pages, d_out_n, d_out_weights, d_freed};
    const dim3 grid((unsigned)n_seq), wg(kEvictThreads);
    if (max_pages <= kEvictThreads) {
        hipLaunchKernelGGL(k_evict<1>, grid, wg, 0, s, A, 1);
    } else if (max_pages <= 4 * kEvictThreads) {
        hipLaunchKernelGGL(k_evict<4>, grid, wg, 0, s, A, 1);
    } else if (max_pages <= 8 * kEvictThreads) {
        hipLaunchKernelGGL(k_evict<8>, grid, wg, 0, s, A, 1);
    } else {
        int64_t parts = max_pages / (4 * kEvictThreads);
        if (parts > 256 / n_seq) parts = 256 / n_seq;
        if (parts < 1) parts = 1;
        hipLaunchKernelGGL(k_evict<0>, dim3((unsigned)(n_seq * parts)), wg, 0, s, A, (int)parts);
    }
    return launch_status();
}

}  // extern "C"
