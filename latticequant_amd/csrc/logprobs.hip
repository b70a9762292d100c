// Log probabilities of given tokens, entropies and top alternatives, from logits, for gfx950.
//
// With c = log2(e), z_i = c x_i - r (one fma; r near the row's largest c x), l = sum 2^z,
// a = sum 2^z z:
//   log p(t) = ln 2 (z_t - log2 l),    H = ln 2 (log2 l - a / l),
// in one pass over the logits: each lane has a reference r of its own, raised (l and a
// rescaled) once the sums show that a logit is far beyond it.
// The `top` largest are a sorted list a wave, an entry a lane.  A lane's vector of logits none
// of which passes the list's last is passed over by one comparison; the others gather in
// LDS, are looked at a logit a lane, and what passes gathers again and goes into the list 64 at
// a time (sorted by a bitonic network, then merged), few of them one by one.  A first bound comes from the workgroup's first vectors: of the four
// largest of the lanes' maxima of every wave the top-th largest, which `top` logits reach.
// Few logits of a row pass it, and most waves need no list.
// Bound by memory with many rows (2048 of 128256 bf16 logits: 82 to 89 us, 6.2 TB/s; with 20
// alternatives 256 rows 23 us), by the latency of a row's loads, lists and sums with one (32000
// logits with 5 alternatives: 9.8 us).
#include <climits>
#include <cmath>

#include "lq_device.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

constexpr int kTop = LQ_LOGPROBS_MAX_TOP;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.0f;
constexpr float kBig = 1e12f;                  // sums beyond it: the reference is too low
constexpr float kHuge = 1e37f;                 // beyond it c x can leave fp32's range
constexpr float kFar = 0x1p20f;                // references beyond it are taken off before the product
constexpr int kUnroll = 4;                     // vectors of 16 bytes a lane has in flight

struct LogArgs {
    const char* logits;
    int64_t stride, vocab;                     // elements
    const int64_t* tokens;
    int top;
    float* logprob;
    float* entropy;
    int64_t* ids;
    float* tops;
};

// A logit and its place as one number: the larger value first (NaN above all; -0 as 0),
// of equal values the lower place.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t at) {
    uint32_t u = __float_as_uint(v + 0.0f);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)(v != v ? 0xffffffffu : u) << 32 | (0xffffffffu - at);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return u == 0xffffffffu ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

template <int DT>
__device__ __forceinline__ float logit(const char* p, int64_t i) {
    if constexpr (DT == LQ_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t u = reinterpret_cast<const uint16_t*>(p)[i];
    return DT == LQ_F16 ? h2f(u) : bf2f(u);
}

// z of a logit by one fma, r = c m rounded: off by that rounding, which all of a row share, so
// it drops out, as long as it is small beside the range of 2^z: 2^-4 at kFar, but 2^9 at a mask of
// -10^10, whose lanes had sums of infinity or 0.  FAR: from the difference (of a
// reference beyond kFar; c x may leave fp32's range), without that rounding
template <bool FAR>
__device__ __forceinline__ float z_of(float x, float m) {
    return FAR ? (x - m) * kLog2e : __builtin_fmaf(x, kLog2e, -(m * kLog2e));
}

struct Stat {
    float m, l, a;                             // reference (of x), sum, sum of 2^z z
};
__device__ __forceinline__ bool far_of(float m) { return fabsf(m) > kFar && fabsf(m) < INFINITY; }
__device__ __forceinline__ float gap(float m, float to) {   // z of one reference from another, as their logits have it
    if (far_of(to)) return far_of(m) ? z_of<true>(m, to) : -__builtin_fmaf(to, kLog2e, -(m * kLog2e));
    return far_of(m) ? z_of<false>(m, to) : m * kLog2e - to * kLog2e;
}
__device__ __forceinline__ void raise(Stat& s, float to) {
    if (s.m == to) return;
    if (s.m == -INFINITY) {                    // nothing but logits of -inf so far
        s.m = to;
        return;
    }
    const float d = gap(s.m, to), f = __builtin_amdgcn_exp2f(d);
    s.a = f == 0.f ? 0.f : f * __builtin_fmaf(d, s.l, s.a);
    s.l *= f;
    s.m = to;
}
// N logits; FAR where the reference is beyond kFar.  Returns their sum: a NaN says that one
// of them is none.
template <bool FAR, int N>
__device__ __forceinline__ float add(Stat& s, const float* x) {
    const float m = s.m == -INFINITY ? 0.f : s.m;
    const float r = -(m * kLog2e);
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        // 2^-200 is 0, as 2^-inf, but 0 times -200 is 0 (and the maximum with a NaN is one)
        const float z = __builtin_elementwise_maximum(FAR ? z_of<true>(x[i], m) : __builtin_fmaf(x[i], kLog2e, r), -200.f);
        const float e = __builtin_amdgcn_exp2f(z);
        l += e;
        s.a = __builtin_fmaf(e, z, s.a);
    }
    s.l += l;
    return l;
}
template <int N>
__device__ __forceinline__ float max_of(const float* x) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) m = fmaxf(fmaxf(m, x[i]), x[i + 1]);   // v_max3
    return N % 2 ? m : fmaxf(m, x[N - 1]);
}

// ---- sorted lists: lane i has the i-th largest of 64 keys, 0 for none

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
    return (uint64_t)dpp<CTRL>((uint32_t)(v >> 32)) << 32 | dpp<CTRL>((uint32_t)v);
}
// the key of lane ^ X
template <int X>
__device__ __forceinline__ uint64_t of_lane_xor(uint64_t k, int lane) {
    if constexpr (X == 1) return dpp<0xB1>(k);           // quad_perm
    if constexpr (X == 2) return dpp<0x4E>(k);
    if constexpr (X == 3) return dpp<0x1B>(k);
    if constexpr (X == 4) return dpp<0x1B>(dpp<0x141>(k));   // row_half_mirror, then each quad reversed
    if constexpr (X == 7) return dpp<0x141>(k);
    if constexpr (X == 8) return dpp<0x128>(k);          // row_ror:8
    if constexpr (X == 15) return dpp<0x140>(k);         // row_mirror
    if constexpr (X == 31) return of_lane_xor<16>(dpp<0x140>(k), lane);
    if constexpr (X == 63) return of_lane_xor<32>(of_lane_xor<31>(k, lane), lane);
    if constexpr (X == 16 || X == 32) {                  // rows (halves) of two registers exchanged
        const uint32_t hi = (uint32_t)(k >> 32), lo = (uint32_t)k;
        if constexpr (X == 16) {
            const auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false), l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
            return lane & 16 ? (uint64_t)h[0] << 32 | l[0] : (uint64_t)h[1] << 32 | l[1];
        } else {
            const auto h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false), l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
            return lane & 32 ? (uint64_t)h[0] << 32 | l[0] : (uint64_t)h[1] << 32 | l[1];
        }
    }
    return 0;
}
// the larger of the keys of lane and lane ^ X in the lower lane
template <int X>
__device__ __forceinline__ uint64_t exchange(uint64_t k, int lane) {
    constexpr int bit = X & ~(X >> 1);                   // X's highest bit
    const uint64_t p = of_lane_xor<X>(k, lane);
    return (p > k) != ((lane & bit) != 0) ? p : k;
}
__device__ __forceinline__ uint64_t halves(uint64_t k, int lane) {   // a bitonic sequence sorted
    k = exchange<32>(k, lane);
    k = exchange<16>(k, lane);
    k = exchange<8>(k, lane);
    k = exchange<4>(k, lane);
    k = exchange<2>(k, lane);
    return exchange<1>(k, lane);
}
__device__ __forceinline__ uint64_t sorted(uint64_t k, int lane) {
    k = exchange<1>(k, lane);
    k = exchange<3>(k, lane);
    k = exchange<1>(k, lane);
    k = exchange<7>(k, lane);
    k = exchange<2>(k, lane);
    k = exchange<1>(k, lane);
    k = exchange<15>(k, lane);
    k = exchange<4>(k, lane);
    k = exchange<2>(k, lane);
    k = exchange<1>(k, lane);
    k = exchange<31>(k, lane);
    k = exchange<8>(k, lane);
    k = exchange<4>(k, lane);
    k = exchange<2>(k, lane);
    k = exchange<1>(k, lane);
    k = exchange<63>(k, lane);
    k = exchange<16>(k, lane);
    k = exchange<8>(k, lane);
    k = exchange<4>(k, lane);
    k = exchange<2>(k, lane);
    return exchange<1>(k, lane);
}
// the 64 largest of a sorted list and another, reversed one
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t reversed, int lane) {
    return halves(a > reversed ? a : reversed, lane);
}

// the top-th largest of 64 numbers, one a lane, none of them a NaN
template <int X>
__device__ __forceinline__ float exchange(float v, int lane) {
    constexpr int bit = X & ~(X >> 1);
    const float p = __uint_as_float((uint32_t)of_lane_xor<X>((uint64_t)__float_as_uint(v), lane));
    return lane & bit ? fminf(v, p) : fmaxf(v, p);
}
__device__ __forceinline__ float nth_largest(float v, int n, int lane) {
    v = exchange<1>(v, lane);
    v = exchange<3>(v, lane);
    v = exchange<1>(v, lane);
    v = exchange<7>(v, lane);
    v = exchange<2>(v, lane);
    v = exchange<1>(v, lane);
    v = exchange<15>(v, lane);
    v = exchange<4>(v, lane);
    v = exchange<2>(v, lane);
    v = exchange<1>(v, lane);
    v = exchange<31>(v, lane);
    v = exchange<8>(v, lane);
    v = exchange<4>(v, lane);
    v = exchange<2>(v, lane);
    v = exchange<1>(v, lane);
    v = exchange<63>(v, lane);
    v = exchange<16>(v, lane);
    v = exchange<8>(v, lane);
    v = exchange<4>(v, lane);
    v = exchange<2>(v, lane);
    v = exchange<1>(v, lane);
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), n - 1));
}

struct List {
    uint64_t key, least;                       // least: entry top - 1
    float bound;                               // no smaller logit is among the `top` largest
    float last;                                // least's value; the bound where there is none yet
    uint64_t* buf;                             // keys that passed, count of them
    int count;
    bool any;                                  // whether the list has any
};
__device__ __forceinline__ void settle(List& t, int top) {
    t.least = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(t.key >> 32), top - 1) << 32 |
              (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)t.key, top - 1);
    t.last = t.least ? key_value(t.least) : t.bound;
}
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// n keys, one a lane and 0 in the others, into the list
__device__ __forceinline__ void take(List& t, uint64_t k, int n, int lane) {
    if (n > 16) {
        t.key = merged(t.key, of_lane_xor<63>(sorted(k, lane), lane), lane);
    } else {
        for (int i = 0; i < n; i++) {
            const uint64_t c = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, i);
            const int at = __builtin_popcountll(__ballot(t.key > c));
            const uint64_t up = dpp<0x138>(t.key);       // wave_shr:1
            t.key = lane < at ? t.key : lane == at ? c : up;
        }
    }
}
__device__ __forceinline__ void flush(List& t, int top, int lane) {   // the buffer's last 64
    const int n = min(t.count, 64);
    t.count -= n;
    wave_lds_sync();
    const uint64_t k = lane < n ? t.buf[t.count + lane] : 0ull;
    wave_lds_sync();
    take(t, k, n, lane);
    settle(t, top);
    t.any = true;
}
// one logit a lane, of those that have one, to the buffer
__device__ __forceinline__ void offer(List& t, float x, uint32_t at, bool mine, int lane) {
    const bool in = mine && !(x < t.last);
    if (!__ballot(in)) return;
    const uint64_t k = key_of(x, at);
    const bool c = in && k > t.least;
    const uint64_t m = __ballot(c);
    if (c) t.buf[t.count + __builtin_popcountll(m & ((1ull << lane) - 1ull))] = k;
    t.count += __builtin_popcountll(m);
}
constexpr int kBuffer = 128;                   // keys left from before and those of an offer
constexpr int kJoint = 512;                    // keys of all waves that go into one list

// (r's rounding is in z and l alike; what it leaves is at most 0 for p = 1, not above)
__device__ __forceinline__ float log_prob(float x, const Stat& s) {
    const float l = __builtin_amdgcn_logf(s.l);
    const bool diff = far_of(s.m) || (fabsf(x) > kHuge && fabsf(x) < INFINITY);
    const float p = diff ? (x - s.m) - kLn2 * l : kLn2 * (z_of<false>(x, s.m) - l);
    return p > 0.f ? 0.f : p;
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, __uint_as_float(dpp<0xB1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp<0x4E>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp<0x141>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp<0x140>(__float_as_uint(v))));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += __uint_as_float(dpp<0xB1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x4E>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x140>(__float_as_uint(v)));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ Stat wave_join(Stat s) {
    raise(s, wave_max(s.m));
    return {s.m, wave_sum(s.l), wave_sum(s.a)};
}

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

// A row a workgroup.
template <int DT, bool TOP, int NW>
__global__ __launch_bounds__(NW * 64) void k_logprobs(LogArgs A) {
    constexpr int E = DT == LQ_F32 ? 4 : 2, V = 16 / E, U = kUnroll, T = NW * 64;
    __shared__ Stat s_stat[NW];
    __shared__ float s_max[64];
    __shared__ int s_count[NW];
    constexpr int M = 64 / V, Q = M + U * 64;  // vectors looked at together, and a wave's queue of them
    __shared__ uint64_t s_key[NW][TOP ? kBuffer : 1], s_joint[TOP ? kJoint : 1];
    __shared__ u4_t s_vec[NW][TOP ? Q : 1];
    __shared__ uint32_t s_at[NW][TOP ? Q : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x, n = A.vocab;
    const char* base = A.logits + row * A.stride * E;
    const int64_t tok = A.tokens ? A.tokens[row] : -1;
    Stat s = {-INFINITY, 0.f, 0.f};
    List t = {0ull, 0ull, -INFINITY, -INFINITY, s_key[wave], 0, false};
    // rows need no alignment: what lies before the first 16-byte boundary and behind the last goes one by one
    const int64_t head = min(n, (int64_t)((16 - ((uintptr_t)base & 15)) & 15) / E);
    const int64_t nv = (n - head) / V, tail = head + nv * V;
    if (wave == 0 && (head || tail < n)) {
        const int64_t i = lane < V ? lane : tail + lane - V;
        const bool mine = lane < V ? i < head : lane < 2 * V && i < n;
        const float x = mine ? logit<DT>(base, i) : -INFINITY;
        raise(s, fmaxf(s.m, x));
        if (mine) {
            if (far_of(s.m)) add<true, 1>(s, &x);
            else add<false, 1>(s, &x);
        }
        if (TOP) offer(t, x, (uint32_t)i, mine, lane);
    }
    int queued = 0;
    auto drain = [&]() __attribute__((always_inline)) {
        wave_lds_sync();
        while (queued) {
            const int m = min(queued, M), at = queued - m + lane / V;
            queued -= m;
            const bool mine = lane / V < m;
            const float x = mine ? logit<DT>(reinterpret_cast<const char*>(&s_vec[wave][at]), lane % V) : 0.f;
            offer(t, x, (uint32_t)head + (mine ? s_at[wave][at] : 0u) * V + lane % V, mine, lane);
            if (t.count >= 64) flush(t, A.top, lane);
        }
        wave_lds_sync();
    };
    u4_t next[U];
    // past the row -inf, which weighs nothing
    constexpr uint32_t none = DT == LQ_F32 ? 0xff800000u : DT == LQ_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    auto fetch = [&](int64_t j0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t j = j0 + u * T + lane;
            next[u] = u4_t{none, none, none, none};
            if (j < nv) next[u] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(base + head * E) + j);
        }
    };
    fetch(wave * 64);
    bool first = TOP;
    for (int64_t j0 = wave * 64; first || j0 < nv; j0 += U * T) {
        u4_t w[U];
        float mx[U];
#pragma unroll
        for (int u = 0; u < U; u++) w[u] = next[u];
        fetch(j0 + U * T);
        auto unpack = [&](const u4_t& v, float* x) __attribute__((always_inline)) {
            if constexpr (DT == LQ_F32) {
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __uint_as_float(v[e]);
            } else {
                unpack8(make_uint4(v[0], v[1], v[2], v[3]), DT, x);
            }
        };
        // Without a look at the largest logit and at -inf first: where the sums show that the
        // reference was too low or is far, or a logit -inf, they are taken again with both.
        float l = 0.f, a = NAN;
        if (j0 >= T) {                         // there is a reference
            const float r = -(s.m * kLog2e);
            a = fabsf(s.m) > kFar ? NAN : 0.f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[V];
                unpack(w[u], x);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float z = __builtin_fmaf(x[e], kLog2e, r), p = __builtin_amdgcn_exp2f(z);
                    l += p;
                    a = __builtin_fmaf(p, z, a);
                }
            }
        }
        if (TOP) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[V];
                unpack(w[u], x);
                mx[u] = max_of<V>(x);
            }
        }
        bool odd = false;                      // a logit is a NaN (or the sum is none for another reason)
        if (__any(!(l < kBig) || a != a)) {
            float x[U * V];
#pragma unroll
            for (int u = 0; u < U; u++) unpack(w[u], x + u * V);
            const float all = max_of<U * V>(x);
            if (all > s.m + kLazy || (s.m == -INFINITY && all > -INFINITY)) raise(s, all);
            l = far_of(s.m) ? add<true, U * V>(s, x) : add<false, U * V>(s, x);
            odd = l != l;
        } else {
            s.l += l;
            s.a += a;
        }
        if (!TOP) continue;
        if (first) {
            first = false;
            constexpr int J = 64 / NW;         // a wave's part of the 64 maxima
            float v = max_of<U>(mx), own = -INFINITY;
            v = v == v ? v : -INFINITY;
            for (int i = 0; i < min(J, A.top); i++) {
                const float b = wave_max(v);
                const int at = __ffsll((long long)__ballot(v == b)) - 1;
                v = lane == at ? -INFINITY : v;
                own = lane == i ? b : own;
            }
            if (lane < J) s_max[wave * J + lane] = own;
            __syncthreads();
            v = s_max[lane];
            if (A.top > 6) {
                t.bound = nth_largest(v, A.top, lane);
            } else {
                for (int i = 0; i < A.top; i++) {
                    t.bound = wave_max(v);
                    const int at = __ffsll((long long)__ballot(v == t.bound)) - 1;
                    v = lane == at ? -INFINITY : v;
                }
            }
            if (!t.least) t.last = t.bound;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t j = j0 + u * T + lane;
            const bool hit = j < nv && (odd || mx[u] >= t.last);
            const uint64_t m = __ballot(hit);
            if (!m) continue;
            if (hit) {
                const int to = queued + __builtin_popcountll(m & ((1ull << lane) - 1ull));
                s_vec[wave][to] = w[u];
                s_at[wave][to] = (uint32_t)j;
            }
            queued += __builtin_popcountll(m);
        }
        if (queued >= M) drain();
    }
    if (TOP && queued) drain();
    s = wave_join(s);
    if (lane == 0) s_stat[wave] = s;
    if (TOP) {
        if (t.any && t.count) flush(t, A.top, lane);
        if (lane == 0) s_count[wave] = t.any ? -1 : t.count;
    }
    __syncthreads();
    int all_n = 0, before = 0;                 // keys of waves without a list
    if (TOP) {
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const int c = max(s_count[w], 0);
            before += w < wave ? c : 0;
            all_n += c;
        }
        const bool lists = all_n > kJoint;     // too many: lists of all waves
        if (lists && !t.any) flush(t, A.top, lane);
        all_n = lists ? 0 : all_n;
        if (t.any) s_key[wave][lane] = t.key;
        else if (lane < t.count) s_joint[before + lane] = t.buf[lane];
        __syncthreads();
        if (wave == 0) {
#pragma unroll 1
            for (int w = 1; w < NW; w++)
                if (lists || s_count[w] < 0) t.key = merged(t.key, s_key[w][63 - lane], lane);
#pragma unroll 1
            for (int i = 0; i < all_n; i += 64)
                take(t, i + lane < all_n ? s_joint[i + lane] : 0ull, min(64, all_n - i), lane);
        }
    }
    if (wave) return;
    s = wave_join(lane < NW ? s_stat[lane] : Stat{-INFINITY, 0.f, 0.f});
    if (lane == 0) {
        A.logprob[row] = tok < 0 ? 0.f : tok >= n ? NAN : log_prob(logit<DT>(base, tok), s);
        const float h = kLn2 * (__builtin_amdgcn_logf(s.l) - s.a / s.l);
        A.entropy[row] = h < 0.f ? 0.f : h;
    }
    if (TOP && lane < A.top) {
        A.ids[row * A.top + lane] = (int64_t)(0xffffffffu - (uint32_t)t.key);
        A.tops[row * A.top + lane] = log_prob(key_value(t.key), s);
    }
}

template <int DT, int NW>
void launch(const LogArgs& A, int64_t rows, hipStream_t s) {
    if (A.top) hipLaunchKernelGGL((k_logprobs<DT, true, NW>), dim3((unsigned)rows), dim3(NW * 64), 0, s, A);
    else hipLaunchKernelGGL((k_logprobs<DT, false, NW>), dim3((unsigned)rows), dim3(NW * 64), 0, s, A);
}
template <int DT>
void launch(const LogArgs& A, int64_t rows, hipStream_t s) {
    // Few rows: a compute unit reads its row as fast as sixteen waves ask for it; with
    // alternatives only one row at a time, by what the waves' queues take of LDS.  bf16, sixteen waves
    // against four, without / with 5 alternatives: 64 x 8192 5.3 / 11.1 us (4.3 / 7.5),
    // 64 x 32000 5.6 / 11.2 (7.8 / 13.0), 256 x 128256 16.3 / 23.3 (23.4 / 36.0), 512 x 128256
    // 25.3 / 42.6 (27.1 / 39.7), 2048 x 128256 88 / 155 (87 / 102).
    if (A.vocab > 16384 && rows <= (A.top ? 256 : 1024)) launch<DT, 16>(A, rows, s);
    else launch<DT, 4>(A, rows, s);
}

}  // namespace

extern "C" {

int lq_token_logprobs(const void *d_logits, int dtype, int64_t stride, int64_t rows, int64_t vocab,
                      const int64_t *d_tokens, int top, float *d_logprob, float *d_entropy, int64_t *d_ids, float *d_top,
                      hipStream_t s) {
    if (!d_logits || dtype < 0 || dtype > 2 || stride < 0 || rows < 1 || rows > INT_MAX || vocab < 1 || vocab > INT_MAX ||
        top < 0 || top > kTop || top > vocab || !d_logprob || !d_entropy || (top && (!d_ids || !d_top)))
        return LQ_ERR_ARG;
    constexpr int64_t kRows = 1 << 22;         // of a launch: a grid has fewer than 2^32 threads
    const char* logits = static_cast<const char*>(d_logits);
    for (int64_t r = 0; r < rows; r += kRows) {
        const LogArgs A = {logits + r * stride * (dtype == LQ_F32 ? 4 : 2), stride, vocab, d_tokens ? d_tokens + r : nullptr, top,
                           d_logprob + r, d_entropy + r, top ? d_ids + r * top : nullptr, top ? d_top + r * top : nullptr};
        const int64_t n = rows - r < kRows ? rows - r : kRows;
        if (dtype == LQ_F32) launch<LQ_F32>(A, n, s);
        else if (dtype == LQ_BF16) launch<LQ_BF16>(A, n, s);
        else launch<LQ_F16>(A, n, s);
    }
    return launch_status();
}

}  // extern "C"
