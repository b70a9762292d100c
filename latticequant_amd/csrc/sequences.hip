// Moves of cached sequences for gfx950: acceptance of drafted tokens, accepted rows
// into the tails, sequences of resident prefixes reordered in place, and new
// prefixes made of chosen sequences and blocks.
#include <climits>
#include <new>

#include "lq_device.h"
#include "lq_readpool.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

// -------------------------------------------------------------- acceptance --

// A logit and its place as one number: the larger value first (NaN above all, as
// torch.argmax orders them; -0 as 0), of equal values the lower place.
__device__ __forceinline__ uint64_t arg_key(float v, uint32_t at) {
    uint32_t u = __float_as_uint(v + 0.0f);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)(v != v ? 0xffffffffu : u) << 32 | (0xffffffffu - at);
}

__device__ __forceinline__ uint64_t key_max(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint64_t wave_key_max(uint64_t k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) k = key_max(k, (uint64_t)__shfl_xor((unsigned long long)k, o, 64));
    return k;
}

template <int DT>
__device__ __forceinline__ float logit(const void* p, int64_t i) {
    if constexpr (DT == LQ_F32) return static_cast<const float*>(p)[i];
    const uint16_t u = static_cast<const uint16_t*>(p)[i];
    return DT == LQ_F16 ? h2f(u) : bf2f(u);
}

// Largest logit of part `blockIdx.x` of row blockIdx.y.  Rows need no alignment: the
// elements before the first 16-byte boundary and after the last go one by one.  Bound by
// memory, each logit read once: 512 rows of 128256 bf16 take 25 us (5.2 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void k_argmax(const char* __restrict__ logits, int64_t sb, int64_t sn, int nodes,
                                                int64_t vocab, int64_t part, uint64_t* __restrict__ keys) {
    constexpr int E = DT == LQ_F32 ? 4 : 2, V = 16 / E;
    __shared__ uint64_t s_k[4];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y, lo = (int64_t)blockIdx.x * part, hi = min(lo + part, vocab);
    const char* base = logits + ((row / nodes) * sb + (row % nodes) * sn) * E;
    float best = -INFINITY;
    int64_t at = lo;
    bool any = false;
    auto take = [&](float v, int64_t i) {   // places grow: the first of equal values stays
        if (!any || v > best || (v != v && best == best)) {
            best = v;
            at = i;
            any = true;
        }
    };
    const int64_t head = min(hi, lo + (int64_t)((16 - ((uintptr_t)(base + lo * E) & 15)) & 15) / E);
    const int64_t nv = (hi - head) / V;
    if (lo + tid < head) take(logit<DT>(base, lo + tid), lo + tid);
    for (int64_t j = tid; j < nv; j += 256) {
        const int64_t i = head + j * V;
        const uint4 w = *reinterpret_cast<const uint4*>(base + i * E);
        float x[8];
        if constexpr (DT == LQ_F32) {
            x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
        } else {
            unpack8(w, DT, x);
        }
#pragma unroll
        for (int e = 0; e < V; e++) take(x[e], i + e);
    }
    const int64_t tail = head + nv * V + tid;
    if (tail < hi) take(logit<DT>(base, tail), tail);
    uint64_t k = wave_key_max(any ? arg_key(best, (uint32_t)at) : 0ull);
    if ((tid & 63) == 0) s_k[tid >> 6] = k;
    __syncthreads();
    if (tid == 0) keys[row * gridDim.x + blockIdx.x] = key_max(key_max(s_k[0], s_k[1]), key_max(s_k[2], s_k[3]));
}

// One wave per sequence: every node's choice (the largest of its parts' keys), then the
// walk, a ballot over the nodes a step.  Bound by latency: 3.9 us for 64 nodes.
__global__ __launch_bounds__(64) void k_accept(const uint64_t* __restrict__ keys, int parts,
                                               const int64_t* __restrict__ given, const int64_t* __restrict__ tokens,
                                               const int32_t* __restrict__ parents, int n, int32_t* __restrict__ path,
                                               int32_t* __restrict__ count, int64_t* __restrict__ next) {
    __shared__ int64_t s_choice[LQ_TREE_MAX_NODES];
    constexpr int Q = LQ_TREE_MAX_NODES / 64;
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.x;
    int par[Q];
    int64_t tok[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const int i = 64 * q + lane;
        par[q] = i < n ? parents[b * n + i] : -2;
        tok[q] = i < n ? tokens[b * n + i] : -1;
        if (i < n) {
            path[b * n + i] = -1;
            if (given) {
                s_choice[i] = given[b * n + i];
            } else {
                uint64_t k = 0;
                for (int p = 0; p < parts; p++) k = key_max(k, keys[(b * n + i) * parts + p]);
                s_choice[i] = (int64_t)(0xffffffffu - (uint32_t)k);
            }
        }
    }
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(par[0]) != -1) {   // node 0 is no root: nothing was drafted here
        if (lane == 0) {
            count[b] = 0;
            next[b] = -1;
        }
        return;
    }
    int cur = 0, steps = 0;
    while (true) {   // a child's number is greater than its parent's: at most n steps
        if (lane == 0) path[b * n + steps] = cur;
        steps++;
        const int64_t want = s_choice[cur];
        int child = -1;
#pragma unroll
        for (int q = Q - 1; q >= 0; q--) {
            const uint64_t hit = __ballot(par[q] == cur && 64 * q + lane > cur && tok[q] == want);
            if (hit) child = 64 * q + __ffsll((long long)hit) - 1;
        }
        if (child < 0) break;
        cur = child;
    }
    if (lane == 0) {
        count[b] = steps;
        next[b] = s_choice[cur];
    }
}

// Parts of a row: enough workgroups for the chip, 4 KB each at least.
int64_t argmax_parts(int64_t rows, int64_t vocab) {
    const int64_t most = (vocab + 2047) / 2048, want = (2048 + rows - 1) / rows;
    return want < most ? want : most;
}

// -------------------------------------------------------------- tail rows --

constexpr int kPairs = 128;   // (destination, source) tensors of one launch

struct RowMoves {
    char* dst[kPairs];
    const char* src[kPairs];
};
struct RowShape {
    int64_t db, dh, dt, sb, sh, st;   // strides in bytes
    int64_t n_seq, heads, cap, rows;  // cap: destination rows; rows: source rows
    int units;                        // 16-byte units of a row
};

// Rows path[b][j], j < count[b], of src behind row len[b] of dst, all tensors of a layout in
// one launch, as a model's layers have the same few rows to move each: up to eight rows of
// a head side by side, 16 bytes a thread.  Bound by latency (3.2 us for 64 tensors of 8
// heads and up to 5 rows, 7.7 us for 16 sequences with up to 27).
__global__ __launch_bounds__(256) void k_append(RowMoves M, RowShape S, int slots, const int32_t* __restrict__ path,
                                                const int32_t* __restrict__ count, const int32_t* __restrict__ len,
                                                int32_t* __restrict__ new_len) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (blockIdx.y == 0 && i < S.n_seq) {
        const int64_t c = min((int64_t)max(count[i], 0), S.rows);
        new_len[i] = (int32_t)min(max((int64_t)len[i], (int64_t)0) + c, S.cap);
    }
    const int u = (int)(i % S.units);
    int64_t k = i / S.units;
    const int j0 = (int)(k % slots);
    k /= slots;
    const int64_t h = k % S.heads, b = k / S.heads;
    if (b >= S.n_seq) return;
    const int64_t n = min((int64_t)max(count[b], 0), S.rows), at = max(len[b], 0);
    char* d = M.dst[blockIdx.y] + b * S.db + h * S.dh + 16 * u;
    const char* s = M.src[blockIdx.y] + b * S.sb + h * S.sh + 16 * u;
    for (int64_t j = j0; j < n && at + j < S.cap; j += slots) {
        const int32_t p = path[b * S.rows + j];
        if (p >= 0 && p < S.rows)
            *reinterpret_cast<uint4*>(d + (at + j) * S.dt) = *reinterpret_cast<const uint4*>(s + (int64_t)p * S.st);
    }
}

// dst[r, h, t] = src[index[r], h, t] for all t < rows
__global__ __launch_bounds__(256) void k_gather(RowMoves M, RowShape S, int64_t n_src,
                                                const int32_t* __restrict__ index) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int u = (int)(i % S.units);
    int64_t k = i / S.units;
    const int64_t t = k % S.rows;
    k /= S.rows;
    const int64_t h = k % S.heads, r = k / S.heads;
    if (r >= S.n_seq) return;
    const int64_t b = min((int64_t)max(index[r], 0), n_src - 1);
    *reinterpret_cast<uint4*>(M.dst[blockIdx.y] + r * S.db + h * S.dh + t * S.dt + 16 * u) =
        *reinterpret_cast<const uint4*>(M.src[blockIdx.y] + b * S.sb + h * S.sh + t * S.st + 16 * u);
}

bool pointers_ok(void* const* dst, const void* const* src, int64_t n) {
    for (int64_t i = 0; i < n; i++)
        if (!dst[i] || !src[i] || ((uintptr_t)dst[i] | (uintptr_t)src[i]) & 15) return false;
    return true;
}

RowMoves moves_of(void* const* dst, const void* const* src, int64_t n) {
    RowMoves m{};
    for (int64_t i = 0; i < n; i++) {
        m.dst[i] = static_cast<char*>(dst[i]);
        m.src[i] = static_cast<const char*>(src[i]);
    }
    return m;
}

// -------------------------------------------------------- resident blocks --

// 16-byte units of a block in each plane, in the order in which a head's units are
// numbered: a, b, mask, scale, meta
constexpr int kUA = 64, kUB = 16, kUM = 2, kUS = 2, kUT = 1, kUnits = kUA + kUB + kUM + kUS + kUT;

struct Planes {
    char *a, *b, *mask, *scale, *meta;
    int64_t cap;   // blocks of a head
};
constexpr int kMaxRes = 64;   // residents of one launch
struct PlaneTable {
    Planes r[kMaxRes];
};

Planes planes_of(const lq_resident* r) {
    return {reinterpret_cast<char*>(r->a), reinterpret_cast<char*>(r->b), reinterpret_cast<char*>(r->mask),
            reinterpret_cast<char*>(r->scale), reinterpret_cast<char*>(r->meta), r->cap_blocks};
}

// Unit w of a head of nb blocks: its plane, the plane's units per block, and its
// place among the plane's units of that head.
struct Unit {
    char* plane;
    int per;
    int64_t at;
};
__device__ __forceinline__ Unit unit_of(const Planes& p, int64_t w, int64_t nb) {
    if (w < nb * kUA) return {p.a, kUA, w};
    w -= nb * kUA;
    if (w < nb * kUB) return {p.b, kUB, w};
    w -= nb * kUB;
    if (w < nb * kUM) return {p.mask, kUM, w};
    w -= nb * kUM;
    if (w < nb * kUS) return {p.scale, kUS, w};
    return {p.meta, kUT, w - nb * kUS};
}

// Workgroups of a head by plane, so that a workgroup's plane is uniform: those of plane p
// end before end[p].
struct Cuts {
    uint32_t end[5];
};
// Where a workgroup works: its plane's unit 0 of head h and block blk0 in sequence 0, the
// bytes from a sequence to the next, its first unit and the plane's units of the head.
struct Part {
    char* at;
    int64_t row;
    uint32_t first, units;
};
__device__ __forceinline__ Part part_of(const Planes& p, const Cuts& c, uint32_t wg, int64_t heads, int64_t h, int64_t blk0,
                                        uint32_t nb, uint32_t threads) {
    const int k = wg < c.end[0] ? 0 : wg < c.end[1] ? 1 : wg < c.end[2] ? 2 : wg < c.end[3] ? 3 : 4;
    const uint32_t per = k == 0 ? kUA : k == 1 ? kUB : k == 2 ? kUM : k == 3 ? kUS : kUT;
    char* base = k == 0 ? p.a : k == 1 ? p.b : k == 2 ? p.mask : k == 3 ? p.scale : p.meta;
    return {base + (h * p.cap + blk0) * per * 16, heads * p.cap * per * 16, (wg - (k ? c.end[k - 1] : 0u)) * threads, nb * per};
}

// In place: a thread has one unit of all sequences and reads the ones that move before it
// writes any.  R: the sequences, at most (their units in registers).  Every load is issued
// before the first wait; where a sequence stays (or its index names none) the load is
// that of one that moves, from cache.  Bound by memory: 8 sequences of 2048 tokens of 64
// prefixes, 1.25 GB read and written, take 255 us (4.9 TB/s); loads that each waited
// for their own took 407.
template <int R>
__global__ __launch_bounds__(256) void k_reorder(PlaneTable P, Cuts cuts, int64_t heads, int n_seq,
                                                 const int32_t* __restrict__ index, int64_t blk0, uint32_t nb) {
    int f[R], any = -1;
#pragma unroll
    for (int s = 0; s < R; s++) f[s] = index[s < n_seq ? s : 0];
#pragma unroll
    for (int s = 0; s < R; s++) {
        if (s >= n_seq || f[s] == s || f[s] < 0 || f[s] >= n_seq) f[s] = -1;
        else any = f[s];
    }
    if (any < 0) return;
    const Part w = part_of(P.r[blockIdx.z], cuts, blockIdx.x, heads, blockIdx.y, blk0, nb, 256);
    const uint32_t u = w.first + threadIdx.x;
    if (u >= w.units) return;
    u32x4_t v[R];   // (a native vector: arrays of the HIP type go through scratch here)
#pragma unroll
    for (int s = 0; s < R; s++) v[s] = reinterpret_cast<const u32x4_t*>(w.at + (f[s] < 0 ? any : f[s]) * w.row)[u];
#pragma unroll
    for (int s = 0; s < R; s++)
        if (f[s] >= 0) reinterpret_cast<u32x4_t*>(w.at + s * w.row)[u] = v[s];
}

// The same for more sequences, their units in LDS (1 KB a sequence and wave; 128 KB are
// taken whatever the number, so one wave a CU: latency-bound, 16 prefixes of 8 heads and 512
// tokens move at 2.0, 2.4, 1.9 and 2.0 TB/s with 17, 32, 64 and 128 sequences, against 6.8
// with 16 in registers).
constexpr int kMaxReorder = 128;
__global__ __launch_bounds__(64) void k_reorder_lds(PlaneTable P, Cuts cuts, int64_t heads, int n_seq,
                                                    const int32_t* __restrict__ index, int64_t blk0, uint32_t nb) {
    __shared__ u32x4_t s_v[kMaxReorder][64];
    const Part w = part_of(P.r[blockIdx.z], cuts, blockIdx.x, heads, blockIdx.y, blk0, nb, 64);
    const uint32_t u = w.first + threadIdx.x;
    if (u >= w.units) return;
    for (int s0 = 0; s0 < n_seq; s0 += 8) {
        u32x4_t v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int s = min(s0 + k, n_seq - 1), f = index[s];
            v[k] = reinterpret_cast<const u32x4_t*>(w.at + (f >= 0 && f < n_seq ? f : s) * w.row)[u];
        }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (s0 + k < n_seq) s_v[s0 + k][threadIdx.x] = v[k];
    }
    for (int s = 0; s < n_seq; s++) {
        const int f = index[s];
        if (f != s && f >= 0 && f < n_seq) reinterpret_cast<u32x4_t*>(w.at + s * w.row)[u] = s_v[s][threadIdx.x];
    }
}

struct Choice {
    const int32_t* index;    // [n_out] sequences
    const int32_t* blocks;   // [n_out][nb] blocks, or null: the first nb
    int64_t n_seq, heads, n_out, nb, src_blocks;
};
// source block (resident head, block) of block j of output head rh = r * heads + h
__device__ __forceinline__ int64_t source_of(const Choice& C, uint32_t rh, uint32_t j, int64_t cap) {
    const uint32_t r = rh / (uint32_t)C.heads, h = rh % (uint32_t)C.heads;
    const int64_t s = min((int64_t)max(C.index[r], 0), C.n_seq - 1);
    const int64_t blk = C.blocks ? min((int64_t)max(C.blocks[r * C.nb + j], 0), C.src_blocks - 1) : (int64_t)j;
    return (s * C.heads + h) * cap + blk;
}

constexpr int kScan = 1024;   // blocks of a scan tile

// A selection's exceptions lie packed, so its first pass scans the chosen blocks' counts:
// k_select_count those of kScan output blocks, each one's sum of those before it in the
// tile (off) and the tile's sum; k_select_bases the tiles' sums.  Both are bound by
// latency (4.8 + 2.0 us for 16384 blocks, 5.6 + 1.8 us for 43232); their total has to reach
// the host, which allocates the list while k_select_planes copies.
__global__ __launch_bounds__(256) void k_select_count(const uint32_t* __restrict__ meta, int64_t cap, Choice C, uint32_t n,
                                                      uint32_t* __restrict__ off, uint32_t* __restrict__ sums) {
    __shared__ uint32_t s_c[kScan], s_w[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t k0 = blockIdx.x * kScan;
#pragma unroll
    for (int i = 0; i < kScan / 256; i++) {
        const uint32_t k = k0 + i * 256 + tid;
        s_c[i * 256 + tid] = k < n ? meta[source_of(C, k / (uint32_t)C.nb, k % (uint32_t)C.nb, cap) * 4 + 3] : 0u;
    }
    __syncthreads();
    const uint4 c = reinterpret_cast<const uint4*>(s_c)[tid];
    const uint32_t mine = c.x + c.y + c.z + c.w;
    uint32_t run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = (uint32_t)__shfl_up((int)run, o, 64);
        if (lane >= o) run += v;
    }
    if (lane == 63) s_w[tid >> 6] = run;
    __syncthreads();
    uint32_t before = run - mine, total = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < (tid >> 6)) before += s_w[w];
        total += s_w[w];
    }
    const uint32_t k = k0 + 4 * tid;
    if (k < n) off[k] = before;
    if (k + 1 < n) off[k + 1] = before + c.x;
    if (k + 2 < n) off[k + 2] = before + c.x + c.y;
    if (k + 3 < n) off[k + 3] = before + c.x + c.y + c.z;
    if (tid == 0) sums[blockIdx.x] = total;
}

// sums[i]: the sum of those before it; the total to n_exc (and to the host).  One wave.
__global__ __launch_bounds__(64) void k_select_bases(uint32_t* sums, int64_t tiles, int32_t* n_exc, int32_t* status,
                                                     int64_t* h_total) {
    const int lane = threadIdx.x;
    uint32_t carry = 0;
    for (int64_t t0 = 0; t0 < tiles; t0 += 64) {
        const uint32_t v = t0 + lane < tiles ? sums[t0 + lane] : 0u;
        uint32_t run = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = (uint32_t)__shfl_up((int)run, o, 64);
            if (lane >= o) run += x;
        }
        if (t0 + lane < tiles) sums[t0 + lane] = carry + run - v;
        carry += (uint32_t)__shfl((int)run, 63, 64);
    }
    if (lane == 0) {
        *n_exc = (int32_t)carry;
        *status = 0;
        if (h_total) *h_total = carry;
    }
}

// The chosen blocks' planes, a 16-byte unit a thread, the metas with their new bases; grid
// (units of a head, output heads).  Bound by memory: 43232 blocks, 59 MB read and as much
// written, 19.8 us (5.9 TB/s).
__global__ __launch_bounds__(256) void k_select_planes(Planes S, Planes D, Choice C, const uint32_t* __restrict__ off,
                                                       const uint32_t* __restrict__ sums) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, rh = blockIdx.y;
    if (i >= (uint32_t)C.nb * kUnits) return;
    const Unit u = unit_of(D, i, C.nb);
    const uint32_t j = (uint32_t)u.at / (uint32_t)u.per, e = (uint32_t)u.at % (uint32_t)u.per, k = rh * (uint32_t)C.nb + j;
    const int64_t from = source_of(C, rh, j, S.cap);
    const char* src = u.plane == D.a ? S.a : u.plane == D.b ? S.b : u.plane == D.mask ? S.mask
                      : u.plane == D.scale ? S.scale : S.meta;
    uint4 w = *reinterpret_cast<const uint4*>(src + (from * u.per + e) * 16);
    if (u.per == kUT) w.z = off[k] + sums[k / kScan];
    *reinterpret_cast<uint4*>(u.plane + ((rh * D.cap + j) * u.per + e) * 16) = w;
}

// exception entries of the chosen blocks, eight lanes a block (3.2 us for 16384 blocks)
__global__ __launch_bounds__(256) void k_select_exc(const uint4* __restrict__ src_meta, const int16_t* __restrict__ src,
                                                    int64_t src_cap, int64_t src_exc, const uint4* __restrict__ dst_meta,
                                                    int16_t* __restrict__ dst, int64_t dst_cap, int64_t dst_exc,
                                                    Choice C, int32_t* status) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, k = i >> 3, rh = k / (uint32_t)C.nb, j = k % (uint32_t)C.nb;
    if (rh >= C.n_out * C.heads) return;
    const uint4 d = dst_meta[rh * dst_cap + j];
    if (!d.w) return;
    const int64_t from = src_meta[source_of(C, rh, j, src_cap)].z;
    for (uint32_t e = i & 7; e < d.w; e += 8) {
        if ((int64_t)d.z + e >= dst_exc) {
            atomicOr(status, LQ_RES_ST_EXC_OVERFLOW);
            return;
        }
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (from + e < src_exc) w = reinterpret_cast<const uint4*>(src)[from + e];
        else atomicOr(status, LQ_RES_ST_EXC_OVERFLOW);   // dropped before already
        reinterpret_cast<uint4*>(dst)[(int64_t)d.z + e] = w;
    }
}

bool res_planes_ok(const lq_resident* r) {
    return r && r->a && r->b && r->mask && r->meta && r->scale && r->n_heads > 0 && r->cap_blocks > 0 &&
           (((uintptr_t)r->a | (uintptr_t)r->b | (uintptr_t)r->mask | (uintptr_t)r->meta | (uintptr_t)r->scale) & 15) == 0;
}

bool choice_of(const lq_resident* src, int64_t n_seq, int64_t src_blocks, const int32_t* index, int64_t n_out,
               const int32_t* blocks, int64_t nb, Choice* c) {
    if (!res_planes_ok(src) || !index || n_seq < 1 || n_out < 1 || n_out > 65535 || nb < 1 || src_blocks < 1 ||
        src->n_heads % n_seq || src_blocks > src->cap_blocks || (!blocks && nb > src_blocks))
        return false;
    *c = {index, blocks, n_seq, src->n_heads / n_seq, n_out, nb, src_blocks};
    return c->heads <= 65535 && n_out * c->heads <= 65535 && nb <= INT_MAX && n_out * c->heads * nb <= (int64_t)INT_MAX / 128;
}
bool takes(const lq_resident* dst, const lq_resident* src, const Choice& c) {
    return res_planes_ok(dst) && dst->a != src->a && dst->n_heads == c.n_out * c.heads && c.nb <= dst->cap_blocks;
}

ReadPool& read_pool() {
    static ReadPool p;   // trivially destroyed: the HIP runtime may be gone by then
    return p;
}

}  // namespace

extern "C" {

int64_t lq_accept_workspace(int64_t n_seq, int64_t n_nodes, int64_t vocab) {
    if (n_seq < 1 || n_nodes < 1 || n_nodes > LQ_TREE_MAX_NODES || vocab < 1 || vocab > INT_MAX ||
        n_seq * n_nodes > 65535)
        return -1;
    return n_seq * n_nodes * argmax_parts(n_seq * n_nodes, vocab) * (int64_t)sizeof(uint64_t);
}

int lq_accept_drafts(const void *d_logits, int dtype, int64_t stride_b, int64_t stride_n, int64_t vocab,
                     const int64_t *d_choice, const int64_t *d_tokens, const int32_t *d_parents, int64_t n_seq,
                     int64_t n_nodes, void *d_work, int64_t work_bytes, int32_t *d_path, int32_t *d_count, int64_t *d_next, hipStream_t s) {
    if ((!d_logits == !d_choice) || !d_tokens || !d_parents || !d_path || !d_count || !d_next || n_seq < 1 ||
        n_seq > INT_MAX || n_nodes < 1 || n_nodes > LQ_TREE_MAX_NODES)
        return LQ_ERR_ARG;
    int64_t parts = 0;
    if (d_logits) {
        if (!d_work || dtype < 0 || dtype > 2 || lq_accept_workspace(n_seq, n_nodes, vocab) < 0 ||
            work_bytes < lq_accept_workspace(n_seq, n_nodes, vocab) || ((uintptr_t)d_work & 7) ||
            ((uintptr_t)d_logits & (dtype == LQ_F32 ? 3 : 1)))
            return LQ_ERR_ARG;
        parts = argmax_parts(n_seq * n_nodes, vocab);
        const int64_t part = ((vocab + parts - 1) / parts + 7) / 8 * 8;
        const dim3 grid((unsigned)parts, (unsigned)(n_seq * n_nodes));
        const char* p = static_cast<const char*>(d_logits);
        uint64_t* keys = static_cast<uint64_t*>(d_work);
        if (dtype == LQ_F32)
            hipLaunchKernelGGL(k_argmax<LQ_F32>, grid, dim3(256), 0, s, p, stride_b, stride_n, (int)n_nodes, vocab, part, keys);
        else if (dtype == LQ_F16)
            hipLaunchKernelGGL(k_argmax<LQ_F16>, grid, dim3(256), 0, s, p, stride_b, stride_n, (int)n_nodes, vocab, part, keys);
        else
            hipLaunchKernelGGL(k_argmax<LQ_BF16>, grid, dim3(256), 0, s, p, stride_b, stride_n, (int)n_nodes, vocab, part, keys);
    }
    hipLaunchKernelGGL(k_accept, dim3((unsigned)n_seq), dim3(64), 0, s, static_cast<const uint64_t*>(d_work), (int)parts,
                       d_choice, d_tokens, d_parents, (int)n_nodes, d_path, d_count, d_next);
    return launch_status();
}

int lq_append_rows(void *const *h_dst, const void *const *h_src, int64_t n, const int64_t *h_dst_stride,
                   const int64_t *h_src_stride, int64_t n_seq, int64_t heads, int64_t cap, int64_t n_nodes,
                   int64_t row_bytes, const int32_t *d_path, const int32_t *d_count, const int32_t *d_len,
                   int32_t *d_new_len, hipStream_t s) {
    if (!h_dst || !h_src || !h_dst_stride || !h_src_stride || n < 1 || n_seq < 1 || heads < 1 || cap < 1 || n_nodes < 1 ||
        n_nodes > LQ_TREE_MAX_NODES || row_bytes < 16 || row_bytes % 16 || row_bytes > 4096 || !d_path || !d_count ||
        !d_len || !d_new_len || cap > INT_MAX)
        return LQ_ERR_ARG;
    const int slots = n_nodes < 8 ? (int)n_nodes : 8;
    const RowShape S = {h_dst_stride[0], h_dst_stride[1], h_dst_stride[2], h_src_stride[0], h_src_stride[1],
                        h_src_stride[2], n_seq, heads, cap, n_nodes, (int)(row_bytes / 16)};
    for (int i = 0; i < 3; i++)
        if (h_dst_stride[i] % 16 || h_src_stride[i] % 16) return LQ_ERR_ARG;
    const int64_t grid = (n_seq * heads * slots * S.units + 255) / 256;
    if (grid > INT_MAX || !pointers_ok(h_dst, h_src, n)) return LQ_ERR_ARG;
    for (int64_t i = 0; i < n; i += kPairs) {
        const int64_t k = n - i < kPairs ? n - i : kPairs;
        const RowMoves m = moves_of(h_dst + i, h_src + i, k);
        hipLaunchKernelGGL(k_append, dim3((unsigned)grid, (unsigned)k), dim3(256), 0, s, m, S, slots, d_path, d_count,
                           d_len, d_new_len);
    }
    return launch_status();
}

int lq_gather_rows(void *const *h_dst, const void *const *h_src, int64_t n, const int64_t *h_dst_stride,
                   const int64_t *h_src_stride, int64_t n_src, int64_t n_out, int64_t heads, int64_t rows,
                   int64_t row_bytes, const int32_t *d_index, hipStream_t s) {
    if (!h_dst || !h_src || !h_dst_stride || !h_src_stride || n < 1 || n_src < 1 || n_out < 1 || heads < 1 || rows < 1 ||
        row_bytes < 16 || row_bytes % 16 || row_bytes > 4096 || !d_index)
        return LQ_ERR_ARG;
    const RowShape S = {h_dst_stride[0], h_dst_stride[1], h_dst_stride[2], h_src_stride[0], h_src_stride[1],
                        h_src_stride[2], n_out, heads, rows, rows, (int)(row_bytes / 16)};
    for (int i = 0; i < 3; i++)
        if (h_dst_stride[i] % 16 || h_src_stride[i] % 16) return LQ_ERR_ARG;
    const int64_t grid = (n_out * heads * rows * S.units + 255) / 256;
    if (grid > INT_MAX || !pointers_ok(h_dst, h_src, n)) return LQ_ERR_ARG;
    for (int64_t i = 0; i < n; i += kPairs) {
        const int64_t k = n - i < kPairs ? n - i : kPairs;
        const RowMoves m = moves_of(h_dst + i, h_src + i, k);
        hipLaunchKernelGGL(k_gather, dim3((unsigned)grid, (unsigned)k), dim3(256), 0, s, m, S, n_src, d_index);
    }
    return launch_status();
}

int lq_resident_reorder(const lq_resident *h_res, int64_t n, int64_t n_seq, const int32_t *d_index, int64_t blk0,
                        int64_t n_blocks, hipStream_t s) {
    if (!h_res || n < 1 || n_seq < 1 || n_seq > kMaxReorder || !d_index || blk0 < 0 || n_blocks < 1) return LQ_ERR_ARG;
    const int64_t n_heads = h_res[0].n_heads;
    for (int64_t i = 0; i < n; i++)
        if (!res_planes_ok(h_res + i) || h_res[i].n_heads != n_heads || n_heads % n_seq ||
            blk0 + n_blocks > h_res[i].cap_blocks)
            return LQ_ERR_ARG;
    const int64_t heads = n_heads / n_seq, wg = n_seq <= 16 ? 256 : 64;
    if (n_blocks > INT_MAX / kUnits || heads > 65535) return LQ_ERR_ARG;
    Cuts cuts;
    const int per[5] = {kUA, kUB, kUM, kUS, kUT};
    uint32_t grid = 0;
    for (int p = 0; p < 5; p++) cuts.end[p] = grid += (uint32_t)((n_blocks * per[p] + wg - 1) / wg);
    for (int64_t i = 0; i < n; i += kMaxRes) {
        const int64_t k = n - i < kMaxRes ? n - i : kMaxRes;
        PlaneTable P{};
        for (int64_t j = 0; j < k; j++) P.r[j] = planes_of(h_res + i + j);
        const dim3 g(grid, (unsigned)heads, (unsigned)k), t((unsigned)wg);
        const uint32_t nb = (uint32_t)n_blocks;
        if (n_seq <= 4) hipLaunchKernelGGL(k_reorder<4>, g, t, 0, s, P, cuts, heads, (int)n_seq, d_index, blk0, nb);
        else if (n_seq <= 8) hipLaunchKernelGGL(k_reorder<8>, g, t, 0, s, P, cuts, heads, (int)n_seq, d_index, blk0, nb);
        else if (n_seq <= 16) hipLaunchKernelGGL(k_reorder<16>, g, t, 0, s, P, cuts, heads, (int)n_seq, d_index, blk0, nb);
        else hipLaunchKernelGGL(k_reorder_lds, g, t, 0, s, P, cuts, heads, (int)n_seq, d_index, blk0, nb);
    }
    return launch_status();
}

int64_t lq_select_workspace(int64_t heads_out, int64_t n_blocks) {
    if (heads_out < 1 || n_blocks < 1 || heads_out > 65535 || heads_out * n_blocks > (int64_t)INT_MAX / 128) return -1;
    const int64_t n = heads_out * n_blocks;
    return (n + (n + kScan - 1) / kScan) * (int64_t)sizeof(uint32_t);
}

int lq_select_count(const lq_resident *src, int64_t n_seq, int64_t src_blocks, const int32_t *d_index, int64_t n_out,
                    const int32_t *d_blocks, int64_t n_blocks, void *d_work, int64_t work_bytes, int32_t *d_n_exc,
                    int32_t *d_status, void **h_read, hipStream_t s) {
    Choice C;
    if (h_read) *h_read = nullptr;
    if (!choice_of(src, n_seq, src_blocks, d_index, n_out, d_blocks, n_blocks, &C) || !d_work || !d_n_exc || !d_status ||
        work_bytes < lq_select_workspace(C.n_out * C.heads, n_blocks) || ((uintptr_t)d_work & 3))
        return LQ_ERR_ARG;
    const int64_t n = C.n_out * C.heads * C.nb, tiles = (n + kScan - 1) / kScan;
    uint32_t* off = static_cast<uint32_t*>(d_work);
    uint32_t* sums = off + n;
    ReadSlot* slot = nullptr;
    if (h_read) {
        slot = new (std::nothrow) ReadSlot;
        if (!slot || !read_pool().take(s, slot)) {
            delete slot;
            return LQ_ERR_LAUNCH;
        }
    }
    hipLaunchKernelGGL(k_select_count, dim3((unsigned)tiles), dim3(256), 0, s, src->meta, src->cap_blocks, C, (uint32_t)n,
                       off, sums);
    hipLaunchKernelGGL(k_select_bases, dim3(1), dim3(64), 0, s, sums, tiles, d_n_exc, d_status, slot ? slot->host : nullptr);
    bool ok = hipGetLastError() == hipSuccess;
    if (slot) {
        ok = hipEventRecord(slot->event, s) == hipSuccess && ok;
        if (ok) {
            *h_read = slot;
        } else {
            (void)hipStreamSynchronize(s);   // no launch may still write the slot
            read_pool().give(*slot);
            delete slot;
        }
    }
    return ok ? LQ_OK : LQ_ERR_LAUNCH;
}

int lq_select_total(void *h_read, int64_t *h_total) {
    if (!h_read) return LQ_ERR_ARG;
    ReadSlot* slot = static_cast<ReadSlot*>(h_read);
    const bool ok = hipEventSynchronize(slot->event) == hipSuccess;
    if (ok && h_total) *h_total = slot->host[0];
    if (ok) read_pool().give(*slot);         // (else a launch may still write it: it is left)
    delete slot;
    return ok ? LQ_OK : LQ_ERR_LAUNCH;
}

int lq_resident_select(const lq_resident *src, int64_t n_seq, int64_t src_blocks, const int32_t *d_index, int64_t n_out,
                       const int32_t *d_blocks, int64_t n_blocks, const lq_resident *dst, const void *d_work,
                       int64_t work_bytes, hipStream_t s) {
    Choice C;
    if (!choice_of(src, n_seq, src_blocks, d_index, n_out, d_blocks, n_blocks, &C) || !takes(dst, src, C) || !d_work ||
        work_bytes < lq_select_workspace(dst->n_heads, n_blocks) || ((uintptr_t)d_work & 3))
        return LQ_ERR_ARG;
    const uint32_t* off = static_cast<const uint32_t*>(d_work);
    hipLaunchKernelGGL(k_select_planes, dim3((unsigned)((C.nb * kUnits + 255) / 256), (unsigned)(C.n_out * C.heads)),
                       dim3(256), 0, s, planes_of(src), planes_of(dst), C, off, off + C.n_out * C.heads * C.nb);
    return launch_status();
}

int lq_resident_select_exceptions(const lq_resident *src, int64_t n_seq, int64_t src_blocks, const int32_t *d_index,
                                  int64_t n_out, const int32_t *d_blocks, int64_t n_blocks, const lq_resident *dst,
                                  hipStream_t s) {
    Choice C;
    if (!choice_of(src, n_seq, src_blocks, d_index, n_out, d_blocks, n_blocks, &C) || !takes(dst, src, C) || !src->exc ||
        !dst->exc || !dst->status || src->exc_cap < 0 || dst->exc_cap < 0)
        return LQ_ERR_ARG;
    const int64_t n = C.n_out * C.heads * C.nb;
    hipLaunchKernelGGL(k_select_exc, dim3((unsigned)((n * 8 + 255) / 256)), dim3(256), 0, s,
                       reinterpret_cast<const uint4*>(src->meta), src->exc, src->cap_blocks, src->exc_cap,
                       reinterpret_cast<const uint4*>(dst->meta), dst->exc, dst->cap_blocks, dst->exc_cap, C, dst->status);
    return launch_status();
}

}  // extern "C"
