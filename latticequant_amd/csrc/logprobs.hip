// Log probabilities of given tokens, entropies and top alternatives, from logits, for gfx950.
//
// With c = log2(e), z_i = c x_i - r (one fma; r near the row's largest c x), l = sum 2^z,
// a = sum 2^z z:
//   log p(t) = ln 2 (z_t - log2 l),    H = ln 2 (log2 l - a / l),
// in one pass over the logits: each lane has a reference r of its own, raised (l and a
// rescaled) once a logit passes it by more than kLazy.  The `top` largest are kept as a
// sorted list a wave, an entry a lane; a logit not above the list's last is passed over by
// the same comparison that guards the reference.
#include <climits>
#include <cmath>

#include "lq_device.h"

using namespace lq;

namespace {

inline int launch_status() { return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_LAUNCH; }

constexpr int kTop = LQ_LOGPROBS_MAX_TOP;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.0f;
constexpr float kHuge = 1e37f;                 // beyond it c x can leave fp32's range

struct LogArgs {
    const char* logits;
    int64_t stride, vocab, part;               // elements
    const int64_t* tokens;
    int top, parts;
    float* logprob;
    float* entropy;
    int64_t* ids;
    float* tops;
    float4* stat;                              // [row][part]: m, l, a
    uint64_t* keys;                            // [row][part][top]
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

// z of a logit: where c x or r would leave fp32's range (a mask of the type's lowest value,
// a row of nothing else) from the difference, else by one fma
template <bool FAR>
__device__ __forceinline__ float z_of(float x, float m) {
    return FAR ? (x - m) * kLog2e : __builtin_fmaf(x, kLog2e, -(m * kLog2e));
}

struct Stat {
    float m, l, a;                             // reference (of x), sum, sum of 2^z z
};
__device__ __forceinline__ bool far_of(float m) { return fabsf(m) > kHuge && fabsf(m) < INFINITY; }
__device__ __forceinline__ float gap(float m, float to) {   // z of one reference from another
    return far_of(m) || far_of(to) ? z_of<true>(m, to) : m * kLog2e - to * kLog2e;
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
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    return {m, a.l + b.l, a.a + b.a};
}

// N logits; FAR where the reference is beyond kHuge.  A sum that is no number says that
// one of them is none.
template <bool FAR, int N>
__device__ __forceinline__ float add(Stat& s, const float x[N]) {
    const float m = s.m == -INFINITY ? 0.f : s.m;
    const float r = -(m * kLog2e);
    float l = 0.f, a = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        // 2^-200 is 0, as 2^-inf, but 0 times -200 is 0 (and the maximum with a NaN is one)
        const float z = __builtin_elementwise_maximum(FAR ? z_of<true>(x[i], m) : __builtin_fmaf(x[i], kLog2e, r), -200.f);
        const float e = __builtin_amdgcn_exp2f(z);
        l += e;
        a = __builtin_fmaf(e, z, a);
    }
    s.l += l;
    s.a += a;
    return l;
}

// The wave's sorted list: lane i has the i-th largest key, 0 where there is none yet.
struct List {
    uint64_t key;
    float last;                                // value of entry top - 1; NaN while there is none
};
__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}
__device__ __forceinline__ void insert(List& t, uint64_t k, int top, int lane) {   // k: wave-uniform
    const int at = __builtin_popcountll(__ballot(t.key > k));
    const uint64_t up = (uint64_t)__shfl_up((unsigned long long)t.key, 1, 64);
    t.key = lane < at ? t.key : lane == at ? k : up;
    const uint64_t l = lane_key(t.key, top - 1);
    t.last = l ? key_value(l) : NAN;
}
// one key a lane, 0 for none
__device__ __forceinline__ void insert_all(List& t, uint64_t k, int top, int lane) {
    for (;;) {
        const uint64_t hit = __ballot(k > lane_key(t.key, top - 1));
        if (!hit) return;
        const int from = __ffsll((long long)hit) - 1;
        insert(t, lane_key(k, from), top, lane);
        if (lane == from) k = 0;
    }
}

// (r's rounding is in z and l alike; what it leaves is at most 0 for p = 1, not above)
__device__ __forceinline__ float log_prob(float x, const Stat& s) {
    const float l = __builtin_amdgcn_logf(s.l);
    const float p = far_of(x) || far_of(s.m) ? (x - s.m) - kLn2 * l : kLn2 * (z_of<false>(x, s.m) - l);
    return p > 0.f ? 0.f : p;
}

template <int DT>
__device__ __forceinline__ void finish(const LogArgs& A, int64_t row, const Stat& s, uint64_t key, int lane) {
    if (lane == 0) {
        const int64_t t = A.tokens ? A.tokens[row] : -1;
        A.logprob[row] = t < 0 ? 0.f : t >= A.vocab ? NAN
                               : log_prob(logit<DT>(A.logits, row * A.stride + t), s);
        const float h = kLn2 * (__builtin_amdgcn_logf(s.l) - s.a / s.l);
        A.entropy[row] = h < 0.f ? 0.f : h;
    }
    if (lane < A.top) {
        A.ids[row * A.top + lane] = (int64_t)(0xffffffffu - (uint32_t)key);
        A.tops[row * A.top + lane] = log_prob(key_value(key), s);
    }
}

// A part of a row a workgroup.
template <int DT, bool TOP>
__global__ __launch_bounds__(kThreads) void k_logprobs(LogArgs A) {
    constexpr int E = DT == LQ_F32 ? 4 : 2, V = 16 / E;
    __shared__ Stat s_stat[kWaves];
    __shared__ uint64_t s_key[kWaves][TOP ? kTop : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (uint32_t)A.parts, part = blockIdx.x % (uint32_t)A.parts;
    const int64_t lo = part * A.part, hi = min(lo + A.part, A.vocab);
    const char* base = A.logits + row * A.stride * E;
    Stat s = {-INFINITY, 0.f, 0.f};
    List t = {0ull, NAN};
    // rows need no alignment: what lies before the first 16-byte boundary and behind the last goes one by one
    const int64_t head = min(hi, lo + (int64_t)((16 - ((uintptr_t)(base + lo * E) & 15)) & 15) / E);
    const int64_t nv = (hi - head) / V, tail = head + nv * V;
    // places grow in a lane's and a wave's order: of equal logits the list keeps the first
    auto single = [&](int64_t i, bool mine) __attribute__((always_inline)) {
        const float x[1] = {mine ? logit<DT>(base, i) : -INFINITY};
        raise(s, fmaxf(s.m, x[0]));
        if (mine) {
            if (far_of(s.m)) add<true, 1>(s, x);
            else add<false, 1>(s, x);
        }
        if (TOP) insert_all(t, mine ? key_of(x[0], (uint32_t)i) : 0ull, A.top, lane);
    };
    if (head > lo) single(lo + tid, lo + tid < head);
    for (int64_t j0 = 0; j0 < nv; j0 += kThreads) {
        const int64_t j = j0 + tid, i = head + j * V;
        const bool mine = j < nv;
        const uint4 w = *reinterpret_cast<const uint4*>(base + (mine ? i : head) * E);
        float x[8];
        if constexpr (DT == LQ_F32) {
            x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
        } else {
            unpack8(w, DT, x);
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < V; e++) mx = fmaxf(mx, x[e]);
        float l = 0.f;
        if (mine) {
            if (mx > s.m + kLazy || (s.m == -INFINITY && mx > -INFINITY)) raise(s, mx);
            l = far_of(s.m) ? add<true, V>(s, x) : add<false, V>(s, x);
        }
        // an equal logit loses to those of earlier rounds, not to all of this one
        const float last = t.last;
        if (TOP && __any(mine && (!(mx <= last) || l != l))) {
#pragma unroll
            for (int e = 0; e < V; e++)
                insert_all(t, mine && !(x[e] <= last) ? key_of(x[e], (uint32_t)(i + e)) : 0ull, A.top, lane);
        }
    }
    if (tail < hi) single(tail + tid, tail + tid < hi);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        s = join(s, {__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.a, o, 64)});
    if (lane == 0) s_stat[wave] = s;
    if (TOP && lane < A.top) s_key[wave][lane] = t.key;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < kWaves; w++) {
        s = join(s, s_stat[w]);
        if (TOP) insert_all(t, lane < A.top ? s_key[w][lane] : 0ull, A.top, lane);
    }
    if (A.parts == 1) {
        finish<DT>(A, row, s, t.key, lane);
        return;
    }
    const int64_t at = row * A.parts + part;
    if (lane == 0) A.stat[at] = make_float4(s.m, s.l, s.a, 0.f);
    if (TOP && lane < A.top) A.keys[at * A.top + lane] = t.key;
}

// A wave per row: its parts joined.
template <int DT, bool TOP>
__global__ __launch_bounds__(64) void k_logprobs_join(LogArgs A) {
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    Stat s = {-INFINITY, 0.f, 0.f};
    for (int p = lane; p < A.parts; p += 64) {
        const float4 x = A.stat[row * A.parts + p];
        s = join(s, {x.x, x.y, x.z});
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        s = join(s, {__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.a, o, 64)});
    List t = {0ull, NAN};
    if (TOP) {
        const int n = A.parts * A.top;
        for (int i = lane; i - lane < n; i += 64)
            insert_all(t, i < n ? A.keys[row * n + i] : 0ull, A.top, lane);
    }
    finish<DT>(A, row, s, t.key, lane);
}

// Parts of a row: enough that all rows' fill the chip, of 8192 logits at least.
int64_t parts_of(int64_t rows, int64_t vocab) {
    const int64_t want = (1024 + rows - 1) / rows, most = (vocab + 8191) / 8192;
    return want < most ? want : most;
}

template <int DT>
void launch(const LogArgs& A, int64_t rows, hipStream_t s) {
    const dim3 grid((unsigned)(rows * A.parts));
    if (A.top) {
        hipLaunchKernelGGL((k_logprobs<DT, true>), grid, dim3(kThreads), 0, s, A);
        if (A.parts > 1) hipLaunchKernelGGL((k_logprobs_join<DT, true>), dim3((unsigned)rows), dim3(64), 0, s, A);
    } else {
        hipLaunchKernelGGL((k_logprobs<DT, false>), grid, dim3(kThreads), 0, s, A);
        if (A.parts > 1) hipLaunchKernelGGL((k_logprobs_join<DT, false>), dim3((unsigned)rows), dim3(64), 0, s, A);
    }
}

}  // namespace

extern "C" {

int64_t lq_logprobs_workspace(int64_t rows, int64_t vocab, int top) {
    if (rows < 1 || rows > INT_MAX / 1024 || vocab < 1 || vocab > INT_MAX || top < 0 || top > kTop || top > vocab) return -1;
    const int64_t parts = parts_of(rows, vocab);
    return parts > 1 ? rows * parts * (16 + 8 * (int64_t)top) : 16;
}

int lq_token_logprobs(const void *d_logits, int dtype, int64_t stride, int64_t rows, int64_t vocab,
                      const int64_t *d_tokens, int top, void *d_work, int64_t work_bytes, float *d_logprob,
                      float *d_entropy, int64_t *d_ids, float *d_top, hipStream_t s) {
    const int64_t need = lq_logprobs_workspace(rows, vocab, top);
    if (!d_logits || dtype < 0 || dtype > 2 || stride < 0 || need < 0 || !d_work || ((uintptr_t)d_work & 15) ||
        work_bytes < need || !d_logprob || !d_entropy || (top && (!d_ids || !d_top)))
        return LQ_ERR_ARG;
    LogArgs A{};
    A.logits = static_cast<const char*>(d_logits);
    A.stride = stride;
    A.vocab = vocab;
    A.parts = (int)parts_of(rows, vocab);
    A.part = (vocab + A.parts - 1) / A.parts;
    A.tokens = d_tokens;
    A.top = top;
    A.logprob = d_logprob;
    A.entropy = d_entropy;
    A.ids = d_ids;
    A.tops = d_top;
    A.stat = static_cast<float4*>(d_work);
    A.keys = reinterpret_cast<uint64_t*>(A.stat + rows * A.parts);
    if (dtype == LQ_F32) launch<LQ_F32>(A, rows, s);
    else if (dtype == LQ_BF16) launch<LQ_BF16>(A, rows, s);
    else launch<LQ_F16>(A, rows, s);
    return launch_status();
}

}  // extern "C"
