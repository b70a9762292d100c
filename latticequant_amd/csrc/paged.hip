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
#include <climits>
#include <cmath>

#include "lq_device.h"
#include "lq_few.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

constexpr int kWaves = 4;                      // of a workgroup
constexpr int kGroups = 512;                   // workgroups at most
constexpr int kMRow = kHd + 4;                 // floats of a piece's row in LDS: o[128], m, l, l32
constexpr int kRecF = 4 + kHd;                 // floats of a record's row: m, l, l32, unused, o[128]
constexpr int kPatch = 8 * 64 * 16;            // bytes of a wave's area for exceptions
constexpr int kThreads = kWaves * 64;

struct Rows {
    const uint16_t* p;
    int64_t sb, sh, st;
};

struct Desc {                                  // the (sequence, head) that a workgroup leaves unfinished
    int32_t unit, more;                        // -1: none; the workgroups that follow it there
};

struct PagedArgs {
    lq_resident k, v;
    const int32_t* pages;
    const int32_t* n_pages;
    const int32_t* tail_len;
    int64_t width, tail_cap;
    Rows q, tk, tv;
    uint16_t* out;
    int64_t ob, oh;
    int n_seq, heads, group, per;              // per: sequences of a lane's sum
    float* rec;                                // [2 workgroup + (0: of an earlier one's, 1: begun here)][row][kRecF]
    Desc* desc;
    float* lse;                                // [unit][row]: m + log2(l32), with the weights' factor 2^kPShift
    float* z;                                  // [unit][page][row]
};

struct Len {
    int pages, tail, tiles, page_tiles;
};
__device__ __forceinline__ Len len_of(const PagedArgs& A, int b) {
    Len l;
    l.pages = min(max(A.n_pages[b], 0), (int)A.width);
    l.tail = A.tail_cap ? (A.tail_len ? min(max(A.tail_len[b], 0), (int)A.tail_cap) : (int)A.tail_cap) : 0;
    l.page_tiles = (l.pages + 1) >> 1;
    l.tiles = l.page_tiles + ((l.tail + 31) >> 5);
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

// K's records as k_tree_few's (KFew), b0 and b1 the tile's blocks
template <bool BIG>
__device__ __forceinline__ void load_k(const lq_resident& r, uint32_t b0, uint32_t b1, uint32_t lane, KFew& d) {
    typedef typename Off<BIG>::type O;
    const uint32_t row = lane & 15, blk = row & 8 ? b1 : b0;
    const uint32_t tok = 8 * ((row >> 2) & 1) + 2 * (row & 3), rec = 16 * (lane >> 4) + tok;
    const O a = (O)blk * 1024 + rec * 4, b = (O)blk * 256 + rec;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        d.a[c] = at<uint2>(r.a, a + 256 * c);
        d.b[c] = at<uint16_t>(r.b, b + 64 * c);
    }
    d.s = at<uint32_t>(r.scale, (O)blk * 32 + tok * 2);
    d.mask = at<uint2>(r.mask, (O)(lane & 4 ? b1 : b0) * 32 + (lane & 3) * 8);
}
// V's: vector lane % 16 of tokens 8 (lane / 16) .. + 7
template <bool BIG>
__device__ __forceinline__ void load_v(const lq_resident& r, uint32_t b0, uint32_t b1, uint32_t lane, Raw& d) {
    typedef typename Off<BIG>::type O;
    const uint32_t blk = lane & 32 ? b1 : b0, rec = 16 * (lane & 15) + 8 * ((lane >> 4) & 1);
    const O a = (O)blk * 1024 + rec * 4;
    d.a[0] = at<uint4>(r.a, a);
    d.a[1] = at<uint4>(r.a, a + 16);
    const uint2 b = at<uint2>(r.b, (O)blk * 256 + rec);
    const uint4 s = at<uint4>(r.scale, (O)blk * 32 + (rec & 15) * 2);
    d.b[0] = b.x;
    d.b[1] = b.y;
    d.s[0] = make_uint2(s.x, s.y);
    d.s[1] = make_uint2(s.z, s.w);
    d.mask[0] = at<uint2>(r.mask, (O)blk * 32 + (rec >> 6) * 8);
}
template <bool BIG>
__device__ __forceinline__ Meta load_meta(const lq_resident& r, uint32_t b0, uint32_t b1, uint32_t lane) {
    typedef typename Off<BIG>::type O;
    const uint4 w = at<uint4>(r.meta, (O)(lane & 32 ? b1 : b0) * 16);
    return {w.x, w.y, w.z, w.w};
}

// Page numbers of a wave's tiles, 64 a register: those of tiles 32 g .. + 31 and of the 32
// behind.  A number outside the pool reads its last page.
struct Pages {
    int32_t near, far, g;
};
__device__ __forceinline__ int32_t load_pages(const int32_t* row, int n, uint32_t cap, int g, int lane) {
    return (int32_t)min((uint32_t)row[min(64 * g + lane, n - 1)], cap - 1);
}
__device__ __forceinline__ uint32_t page_of(const Pages& p, int j) {   // j: the page's place, within the two
    const int at = j & 63;
    return (uint32_t)((j >> 6) == p.g ? __builtin_amdgcn_readlane(p.near, at) : __builtin_amdgcn_readlane(p.far, at));
}

__device__ __forceinline__ float pair_sum(float v) {   // of lane and lane ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// few_attend; with SUMS also the logarithm (base 2) of the sum of the lane's page (lanes
// 0..31 hold the first page's tokens, 32..63 the second's), and the row's sum l32, both of
// the weights in 32 bits, as they are before they are rounded for P V.
template <bool SUMS>
__device__ __forceinline__ float attend(f4_t s[2], uint32_t word, bool every, const uint32_t vp[4][8], int lane,
                                        FewState& st, float& l32) {
    if constexpr (!SUMS) {
        few_attend(s, word, every, vp, lane, st);
        return 0.f;
    }
    const float was = st.m, off = few_reference(s, word, every, lane, st);
    if (was != st.m) l32 *= __builtin_amdgcn_exp2f(was - st.m);
    uint32_t p[4];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], kScale2, off));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][i], kScale2, off));
        p[i] = pair_h(x, y);
        st.l = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, p[i]), h2_t{(_Float16)1.f, (_Float16)1.f}, st.l, false);
        sum += x + y;
    }
    few_products(p, vp, st);
    l32 += sum;
    return __builtin_amdgcn_logf(pair_sum(sum)) - off + kPShift;
}

__device__ __forceinline__ void zero_out(const PagedArgs& A, int b, int tid) {
    const int n = A.heads * A.group * (kHd / 8);
    for (int i = tid; i < n; i += kThreads)
        *reinterpret_cast<uint4*>(A.out + b * A.ob + (i >> 4) * A.oh + 8 * (i & 15)) = make_uint4(0u, 0u, 0u, 0u);
}

template <bool BF16>
__device__ __forceinline__ void put8(const PagedArgs& A, int unit, int row, int d, const float x[8], float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float u = x[2 * i] * inv, v = x[2 * i + 1] * inv;
        w[i] = BF16 ? (uint32_t)f2bf(u) | ((uint32_t)f2bf(v) << 16) : pair_h(u, v);
    }
    const int b = unit / A.heads, h = unit % A.heads;
    *reinterpret_cast<uint4*>(A.out + b * A.ob + (int64_t)(h * A.group + row) * A.oh + d) = make_uint4(w[0], w[1], w[2], w[3]);
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
    return l;
}
template <bool BF16, bool SUMS, bool BIG>
__global__ __launch_bounds__(kThreads, 2) void k_paged(PagedArgs A) {
    extern __shared__ __align__(16) char s_dyn[];
    // pieces in the order of the list: wave w's first (2 w), which ends its unit there, and its last (2 w + 1)
    __shared__ int s_unit[2 * kWaves], s_begins[2 * kWaves];
    __shared__ uint32_t s_end;                 // where the list's unit that is begun here and not ended ends
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4, G = A.group;
    const int slot = G * kMRow * 4;            // bytes of a piece
    const int last_area = max(kPatch, slot), stride = last_area + slot;
    char* mine = s_dyn + wave * stride;        // exceptions, then the wave's last piece; behind it its first
    u32x4_t* area = reinterpret_cast<u32x4_t*>(mine);

    // ---- the workgroup's share of the list, found by every wave for itself
    Lens lens = {0, 0};
    uint32_t own = 0;
    for (int b = lane * A.per; b < min((lane + 1) * A.per, A.n_seq); b++) {
        const Len l = len_of(A, b);
        lens = {l.pages, l.tail};
        own += (uint32_t)l.tiles * A.heads;
    }
    uint32_t upto = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(upto, o, 64);
        upto += lane >= o ? x : 0u;
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63), before = upto - own;
    if (tid < 2 * kWaves) s_unit[tid] = -1;
    __syncthreads();
    for (int b = blockIdx.x; b < A.n_seq; b += gridDim.x)
        if (len_at(A, lens, b).tiles == 0) zero_out(A, b, tid);
    const uint32_t groups = max(1u, min((uint32_t)gridDim.x, (total + kWaves - 1) / kWaves));
    const uint32_t me = blockIdx.x;
    if (me >= groups) {
        if (tid == 0) A.desc[me] = {-1, 0};
        return;
    }
    const uint32_t lo = (uint32_t)((uint64_t)me * total / groups), hi = (uint32_t)((uint64_t)(me + 1) * total / groups);
    uint32_t pos = lo + (uint32_t)((uint64_t)(hi - lo) * wave / kWaves);
    const uint32_t end = lo + (uint32_t)((uint64_t)(hi - lo) * (wave + 1) / kWaves);

    if (pos < end) {
        const uint64_t there = __ballot(pos >= before && pos - before < own);
        const int from = __ffsll((long long)there) - 1;
        uint32_t rem = pos - (uint32_t)__builtin_amdgcn_readlane((int)before, from);
        int b = from * A.per;
        Len L = len_at(A, lens, b);
        for (int k = 1; k < A.per; k++) {
            const uint32_t n = (uint32_t)L.tiles * A.heads;
            if (rem < n || b + 1 >= A.n_seq) break;
            rem -= n;
            L = len_of(A, ++b);
        }
        const uint32_t tiles = (uint32_t)max(L.tiles, 1);
        int h = (int)(rem / tiles), t = (int)(rem % tiles);
        for (;;) {
            const int unit = b * A.heads + h;
            const int n = (int)min((uint32_t)(L.tiles - t), end - pos);
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
            float l32 = 0.f;
#pragma unroll
            for (int mm = 0; mm < 8; mm++) st.o[mm] = f4_t{0.f, 0.f, 0.f, 0.f};

            // ---- the pages' tiles
            const int pe = min(t + n, L.page_tiles);
            if (t < pe) {
                const int32_t* row = A.pages + b * A.width;
                const uint32_t cap = (uint32_t)A.k.cap_blocks, hb = (uint32_t)h * cap, hbv = (uint32_t)h * (uint32_t)A.v.cap_blocks;
                Pages pg;
                pg.g = t >> 5;
                pg.near = load_pages(row, L.pages, cap, pg.g, lane);
                pg.far = load_pages(row, L.pages, cap, pg.g + 1, lane);
                KFew kr;
                Raw vr;
                Meta mk, mv, nk, nv;
                uint4 ek, ev;
                const auto blocks = [&](int tile, uint32_t& x, uint32_t& y) __attribute__((always_inline)) {
                    const int j = 2 * min(tile, pe - 1);
                    x = page_of(pg, j);
                    y = page_of(pg, min(j + 1, L.pages - 1));
                };
                {
                    uint32_t x, y;
                    blocks(t, x, y);
                    mk = load_meta<BIG>(A.k, hb + x, hb + y, lane);
                    mv = load_meta<BIG>(A.v, hbv + x, hbv + y, lane);
                    load_k<BIG>(A.k, hb + x, hb + y, lane, kr);
                    load_v<BIG>(A.v, hbv + x, hbv + y, lane, vr);
                    blocks(t + 1, x, y);
                    nk = load_meta<BIG>(A.k, hb + x, hb + y, lane);
                    nv = load_meta<BIG>(A.v, hbv + x, hbv + y, lane);
                    ek = load_entry(A.k, mk, lane);
                    ev = load_entry(A.v, mv, lane);
                }
                for (int tile = t; tile < pe; tile++) {
                    const uint32_t word = 2 * tile + 1 < L.pages ? ~0u : 0xffffu;
                    f4_t s[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
                    uint32_t vp[4][8], p[8][4];
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
                        s[j & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(p[j][0], p[j][1], p[j][2], p[j][3]), q[j >> 1],
                                                                          s[j & 1], 0, 0, 0);
                    }
                    decode_v(vr, vp);
                    if (const uint32_t most = most_of(mv)) patch_v(A.v, vr, mv, ev, most, lane, area, vp);
                    scale_v(vr, word, lane, vp);
                    __builtin_amdgcn_sched_barrier(0);   // every use of the records before their reload
                    // the next tile's records and the bases of the one behind; past the end the last again
                    ek = load_entry(A.k, nk, lane);
                    ev = load_entry(A.v, nv, lane);
                    mk = nk;
                    mv = nv;
                    uint32_t x, y;
                    if (((tile + 1) >> 5) != pg.g) {
                        pg.g++;
                        pg.near = pg.far;
                        pg.far = load_pages(row, L.pages, cap, pg.g + 1, lane);
                    }
                    blocks(tile + 1, x, y);
                    load_k<BIG>(A.k, hb + x, hb + y, lane, kr);
                    load_v<BIG>(A.v, hbv + x, hbv + y, lane, vr);
                    blocks(tile + 2, x, y);
                    nk = load_meta<BIG>(A.k, hb + x, hb + y, lane);
                    nv = load_meta<BIG>(A.v, hbv + x, hbv + y, lane);
                    const float z = attend<SUMS>(s, word, word == ~0u, vp, lane, st, l32);
                    if (SUMS) {
                        const int j = 2 * tile + (lane >> 5);
                        if (!(g & 1) && col < G && j < L.pages) A.z[((int64_t)unit * A.width + j) * G + col] = z;
                    }
                }
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
                rows_v<BF16>(A.tv.p + b * A.tv.sb + h * A.tv.sh, A.tv.st, t0, have, word, lane, vp);
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        s[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            __builtin_bit_cast(h8_t, BF16 ? bf_to_h(w[y][c]) : w[y][c]), q[c], s[y], 0, 0, 0);
                attend<SUMS>(s, word, word == ~0u, vp, lane, st, l32);
            }
            // ---- the unit is written out, or its piece kept
            float l = st.l + __shfl_xor(st.l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            if (SUMS) {
                l32 += __shfl_xor(l32, 16, 64);
                l32 += __shfl_xor(l32, 32, 64);
            }
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
                    if (SUMS && g == 0) A.lse[(int64_t)unit * G + col] = st.m + __builtin_amdgcn_logf(l32);
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
                    if (!ends && pos + n == hi) s_end = pos + (uint32_t)(L.tiles - t);
                }
            }
            pos += n;
            if (pos == end) break;
            t = 0;
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

    // ---- pieces joined: 16 lanes a row, eight dimensions a lane
    Desc left = {-1, 0};
    const int row = tid >> 4, d = 8 * (tid & 15);
    for (int i = 0; i < 2 * kWaves;) {
        const int unit = s_unit[i];
        if (unit < 0) {
            i++;
            continue;
        }
        const bool begins = s_begins[i] != 0;
        bool ends = false;
        float m = -INFINITY, l = 0.f, l32 = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (; i < 2 * kWaves && (s_unit[i] == unit || s_unit[i] < 0); i++) {
            if (s_unit[i] < 0) continue;
            ends = !(i & 1);
            if (row >= G) continue;
            const float* p = reinterpret_cast<const float*>(s_dyn + (i >> 1) * stride + (ends ? last_area : 0)) + row * kMRow;
            const float pm = p[kHd], M = fmaxf(m, pm);
            const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M);
            const float f1 = pm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(pm - M);
            l = l * f0 + p[kHd + 1] * f1;
            if (SUMS) l32 = l32 * f0 + p[kHd + 2] * f1;
            const f4_t u = *reinterpret_cast<const f4_t*>(p + d), v = *reinterpret_cast<const f4_t*>(p + d + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = x[e] * f0 + u[e] * f1;
                x[4 + e] = x[4 + e] * f0 + v[e] * f1;
            }
            m = M;
        }
        if (begins && ends) {
            if (row < G) {
                put8<BF16>(A, unit, row, d, x, 1.f / l);
                if (SUMS && d == 0) A.lse[(int64_t)unit * G + row] = m + __builtin_amdgcn_logf(l32);
            }
        } else {
            if (row < G) {
                float* rec = A.rec + ((int64_t)(2 * me + (begins ? 1 : 0)) * G + row) * kRecF;
                *reinterpret_cast<f4_t*>(rec + 4 + d) = f4_t{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<f4_t*>(rec + 8 + d) = f4_t{x[4], x[5], x[6], x[7]};
                if (d == 0) *reinterpret_cast<f4_t*>(rec) = f4_t{m, l, l32, 0.f};
            }
            if (begins) left = {unit, (int32_t)(((uint64_t)s_end * groups - 1) / total - me)};
        }
    }
    if (tid == 0) A.desc[me] = left;
}

// The records of a unit that several workgroups share, a workgroup per row: thread
// (sub, dq) sums dimensions 4 dq .. + 3 of records sub, sub + 8, .., then the eight sums
// are joined in order.
template <bool BF16, bool SUMS>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs A) {
    constexpr int kUp = 8;                     // records in flight per thread
    __shared__ __align__(16) f4_t s_o[8][32];
    __shared__ float s_m[8], s_l[8], s_l32[8];
    const int dq = threadIdx.x & 31, sub = threadIdx.x >> 5, row = blockIdx.y, wg = blockIdx.x;
    const Desc D = A.desc[wg];
    if (D.unit < 0) return;
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
#pragma unroll
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
    if (SUMS && lane == 0) A.lse[(int64_t)D.unit * A.group + row] = M + __builtin_amdgcn_logf(L32);
}

// weights[b][j] = decay * weights[b][j] + the page's weight of this step (decay 0: that
// alone), a lane a page, the heads dealt to four waves whose sums are joined in order.
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

// A sequence a workgroup: the room-th largest weight of the pages that may go, by a radix
// search of 11, 11 and 10 bits, then one pass in the order of the pages, each wave a part.
__global__ __launch_bounds__(kEvictThreads) void k_evict(EvictArgs A) {
    __shared__ uint32_t s_bin[kBins];
    __shared__ uint32_t s_part[kEvictWaves];
    __shared__ uint32_t s_pick, s_left;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t at = blockIdx.x * A.width;
    const int n = min(max(A.n_pages[blockIdx.x], 0), (int)A.width);
    const int lo = min(A.sink, n), hi = max(lo, n - A.recent);
    const bool all = n <= A.keep;
    uint32_t room = all ? 0u : (uint32_t)max(0, A.keep - lo - (n - hi));
    const uint32_t kept_n = all ? (uint32_t)n : (uint32_t)lo + (uint32_t)(n - hi) + room;
    uint32_t prefix = 0;                       // the bits found so far
    if (!all && room) {
        for (int digit = 0; digit < 3; digit++) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
            for (int i = tid; i < kBins; i += kEvictThreads) s_bin[i] = 0u;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += kEvictThreads) {
                const uint32_t k = weight_key(A.weights[at + j]);
                if (digit == 0 || k >> (shift + bits) == prefix) atomicAdd(&s_bin[(k >> shift) & ((1u << bits) - 1u)], 1u);
            }
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
            for (int w = 0; w < wave; w++) upto += s_part[w];
            const uint32_t before = upto - c0 - c1;
            if (before < room && room <= upto) {
                const bool second = room > before + c0;
                s_pick = (uint32_t)(kBins - 1 - 2 * tid - (second ? 1 : 0));
                s_left = room - before - (second ? c0 : 0u);
            }
            __syncthreads();
            prefix = prefix << bits | s_pick;
            room = s_left;
            __syncthreads();
        }
    }
    // kept: the protected, what is above the key, and the first `room` of those equal to it
    const int seg = ((n + 63) / 64 + kEvictWaves - 1) / kEvictWaves * 64;
    const int j0 = wave * seg, j1 = min(n, j0 + seg);
    const bool some = !all && kept_n > (uint32_t)(lo + n - hi);
    uint32_t ties = 0, above = 0;
    for (int j = j0; j < j1; j += 64) {
        const int i = j + lane;
        const bool open = i >= lo && i < hi;
        const uint32_t k = open && i < j1 ? weight_key(A.weights[at + i]) : 0u;
        ties += __builtin_popcountll(__ballot(open && i < j1 && some && k == prefix));
        above += __builtin_popcountll(__ballot(i < j1 && (all || !open || (some && k > prefix))));
    }
    if (lane == 0) {
        s_bin[wave] = ties;
        s_bin[kEvictWaves + wave] = above;
    }
    __syncthreads();
    uint32_t tie = 0, to = 0;                  // equal and kept ones before the wave's part
    for (int w = 0; w < wave; w++) {
        to += s_bin[kEvictWaves + w] + min(s_bin[w], tie < room ? room - tie : 0u);
        tie += s_bin[w];
    }
    for (int j = j0; j < j1; j += 64) {
        const int i = j + lane;
        const bool in = i < j1, open = i >= lo && i < hi;
        const float w = in ? A.weights[at + i] : 0.f;
        const int32_t page = in ? A.pages[at + i] : 0;
        const uint32_t k = weight_key(w);
        const uint64_t eq = __ballot(in && open && some && k == prefix), below = (1ull << lane) - 1ull;
        const bool keep = in && (all || !open || (some && (k > prefix || (k == prefix && tie + __builtin_popcountll(eq & below) < room))));
        const uint64_t kept = __ballot(keep);
        const uint32_t p = to + __builtin_popcountll(kept & below);
        if (keep) {
            A.out_pages[at + p] = page;
            A.out_weights[at + p] = w;
        } else if (in) {
            A.freed[at + (uint32_t)i - p] = page;
        }
        tie += __builtin_popcountll(eq);
        to += __builtin_popcountll(kept);
    }
    for (int64_t j = kept_n + tid; j < A.width; j += kEvictThreads) {
        A.out_pages[at + j] = -1;
        A.out_weights[at + j] = 0.f;
    }
    for (int64_t j = n - kept_n + tid; j < A.width; j += kEvictThreads) A.freed[at + j] = -1;
    if (tid == 0) A.out_n[blockIdx.x] = (int32_t)kept_n;
}

// ------------------------------------------------------------------- plan --

struct Plan {
    int grid;
    int64_t rec, desc, lse, z, bytes;          // bytes before each, and in all
};
bool plan(int64_t n_seq, int64_t heads, int64_t group, int64_t width, int64_t tail_cap, bool weights, Plan* p) {
    if (n_seq < 1 || heads < 1 || group < 1 || group > 16 || width < 0 || tail_cap < 0 || width > INT_MAX / 64 ||
        tail_cap > INT_MAX / 64 || n_seq > 65535 || heads > 65535 || n_seq * heads > INT_MAX / 16)
        return false;
    const int64_t tiles = (width + 1) / 2 + (tail_cap + 31) / 32;
    if (tiles > INT_MAX / (n_seq * heads)) return false;
    const int64_t most = (n_seq * heads * tiles + kWaves - 1) / kWaves;
    p->grid = (int)(most < 1 ? 1 : most < kGroups ? most : kGroups);
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    p->rec = 0;
    p->desc = p->rec + up(2 * p->grid * group * kRecF * 4);
    p->lse = p->desc + up(p->grid * (int64_t)sizeof(Desc));
    p->z = p->lse + (weights ? up(n_seq * heads * group * 4) : 0);
    p->bytes = p->z + (weights ? up(n_seq * heads * group * width * 4) : 0);
    return true;
}

bool pool_ok(const lq_resident* r) {
    return r && r->a && r->b && r->mask && r->meta && r->scale && r->n_heads > 0 && r->cap_blocks > 0 && r->exc_cap >= 0 &&
           r->cap_blocks <= INT_MAX / r->n_heads;
}
bool rows_ok(const lq_rows* r) {
    return r && r->p && ((uintptr_t)r->p & 15) == 0 && r->stride_b % 8 == 0 && r->stride_h % 8 == 0 && r->stride_t % 8 == 0;
}
Rows rows_of(const lq_rows* r) { return {static_cast<const uint16_t*>(r->p), r->stride_b, r->stride_h, r->stride_t}; }

template <bool BF16, bool SUMS>
void paged_launch(const PagedArgs& A, int grid, bool big, hipStream_t s) {
    const int slot = A.group * kMRow * 4;
    const size_t lds = (size_t)kWaves * ((slot > kPatch ? slot : kPatch) + slot);
    if (big) hipLaunchKernelGGL((k_paged<BF16, SUMS, true>), dim3((unsigned)grid), dim3(kThreads), lds, s, A);
    else hipLaunchKernelGGL((k_paged<BF16, SUMS, false>), dim3((unsigned)grid), dim3(kThreads), lds, s, A);
    if (grid > 1) hipLaunchKernelGGL((k_paged_join<BF16, SUMS>), dim3((unsigned)grid, (unsigned)A.group), dim3(256), 0, s, A);
}

}  // namespace

extern "C" {

int64_t lq_paged_attn_workspace(int64_t n_seq, int64_t heads, int group, int64_t max_pages, int64_t tail_cap, int weights) {
    Plan p;
    return plan(n_seq, heads, group, max_pages, tail_cap, weights != 0, &p) ? p.bytes : -1;
}

int lq_paged_attention(const lq_resident *k, const lq_resident *v, const lq_rows *q, int64_t n_seq, int group,
                       const int32_t *d_pages, int64_t max_pages, const int32_t *d_n_pages, const lq_rows *tail_k,
                       const lq_rows *tail_v, int64_t tail_cap, const int32_t *d_tail_len, float *d_weights, float decay,
                       int dtype, void *d_work, int64_t work_bytes, const lq_rows *out, hipStream_t s) {
    if (!pool_ok(k) || !pool_ok(v) || k->n_heads != v->n_heads || k->cap_blocks != v->cap_blocks || !rows_ok(q) ||
        !rows_ok(out) || !d_n_pages || (max_pages > 0 && !d_pages) || !d_work || ((uintptr_t)d_work & 15) ||
        (dtype != LQ_F16 && dtype != LQ_BF16))
        return LQ_ERR_ARG;
    if (tail_cap > 0 && (!rows_ok(tail_k) || !rows_ok(tail_v))) return LQ_ERR_ARG;
    Plan p;
    if (!plan(n_seq, k->n_heads, group, max_pages, tail_cap, d_weights != nullptr, &p) || work_bytes < p.bytes)
        return LQ_ERR_ARG;
    PagedArgs A{};
    A.k = *k;
    A.v = *v;
    // an empty exception list is read at its first entry and the value not used
    if (!A.k.exc || A.k.exc_cap == 0) A.k.exc = reinterpret_cast<int16_t*>(A.k.a);
    if (!A.v.exc || A.v.exc_cap == 0) A.v.exc = reinterpret_cast<int16_t*>(A.v.a);
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
    A.heads = (int)k->n_heads;
    A.group = group;
    A.per = (int)((n_seq + 63) / 64);
    char* w = static_cast<char*>(d_work);
    A.rec = reinterpret_cast<float*>(w + p.rec);
    A.desc = reinterpret_cast<Desc*>(w + p.desc);
    A.lse = reinterpret_cast<float*>(w + p.lse);
    A.z = reinterpret_cast<float*>(w + p.z);
    const bool big = k->n_heads * k->cap_blocks > (int64_t)(UINT32_MAX / 1024);
    if (dtype == LQ_BF16) {
        if (d_weights) paged_launch<true, true>(A, p.grid, big, s);
        else paged_launch<true, false>(A, p.grid, big, s);
    } else {
        if (d_weights) paged_launch<false, true>(A, p.grid, big, s);
        else paged_launch<false, false>(A, p.grid, big, s);
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
        n_seq > INT_MAX || max_pages < 1 || max_pages > INT_MAX / 2 || sink < 0 || recent < 0 || sink > INT_MAX / 4 ||
        recent > INT_MAX / 4 || keep < sink + recent || keep > INT_MAX)
        return LQ_ERR_ARG;
    const EvictArgs A = {d_pages, d_n_pages, d_weights, max_pages, (int)keep, (int)sink, (int)recent,
                         d_out_pages, d_out_n, d_out_weights, d_freed};
    hipLaunchKernelGGL(k_evict, dim3((unsigned)n_seq), dim3(kEvictThreads), 0, s, A);
    return launch_status();
}

}  // extern "C"
