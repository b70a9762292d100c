// Records of the resident form (layout in latticequant_amd.h) as fp16 operands,
// shared by the kernels that read it.
#pragma once

#include "lq_device.h"

namespace lq {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kHd = 128;
constexpr int kRB = 16;                       // tokens per resident block
constexpr uint32_t kPairBias = 0x60206020u;   // fp16 pair (528, 528)
constexpr uint32_t kFieldMask = 0x003E003Eu;  // bits 1..5 of both halves
constexpr uint32_t kLsbMask = 0x08420842u;    // low bits of u0..u5 in the a word

__device__ __forceinline__ uint32_t unbias(uint32_t v) {
    const h2_t r = __builtin_bit_cast(h2_t, v) - __builtin_bit_cast(h2_t, kPairBias);
    return __builtin_bit_cast(uint32_t, r);
}

// One record -> four fp16 pairs 528 + c of coordinates (0,1) (2,3) (4,5) (6,7).
__device__ __forceinline__ void rec_pairs(uint32_t a, uint32_t b, uint32_t p[4]) {
    // (coset bit at bit 0 and 16) | 0x60006000: byte 0 of a copied to byte 2
    // by one byte permute, then one AND-OR (a select between two constants
    // would take three instructions)
    const uint32_t kc = (__builtin_amdgcn_perm(0u, a, 0x0c000c00u) & 0x00010001u) | 0x60006000u;
    p[0] = (a & kFieldMask) | kc;
    p[1] = ((a >> 5) & kFieldMask) | kc;
    p[2] = ((a >> 10) & kFieldMask) | kc;
    const uint32_t c7h = ((b >> 5) & 7u) | ((a >> 13) & 8u);
    const uint32_t par = ((uint32_t)__builtin_popcount(a & kLsbMask) + b) & 1u;
    const uint32_t u7 = (c7h << 1) | par;
    p[3] = kc | ((b & 31u) << 1) | (u7 << 17);
}

// Records of tokens t and t+1 (same vector) -> eight fp16 pairs
// (coordinate i of t, coordinate i of t+1), values 528 + c.
__device__ __forceinline__ void rec_pairs_tok(uint32_t a0, uint32_t b0, uint32_t a1, uint32_t b1, uint32_t p[8]) {
    const uint32_t lo = __builtin_amdgcn_perm(a1, a0, 0x05040100u);   // a0[15:0] | a1[15:0] << 16
    const uint32_t hi = __builtin_amdgcn_perm(a1, a0, 0x07060302u);   // a0[31:16] | a1[31:16] << 16
    const uint32_t kc = 0x60006000u | (lo & 0x00010001u);             // coset of t at bit 0, of t+1 at bit 16
    p[0] = (lo & kFieldMask) | kc;
    p[2] = ((lo >> 5) & kFieldMask) | kc;
    p[4] = ((lo >> 10) & kFieldMask) | kc;
    p[1] = (hi & kFieldMask) | kc;
    p[3] = ((hi >> 5) & kFieldMask) | kc;
    p[5] = ((hi >> 10) & kFieldMask) | kc;
    const uint32_t h0 = ((b0 >> 5) & 7u) | ((a0 >> 13) & 8u);
    const uint32_t h1 = ((b1 >> 5) & 7u) | ((a1 >> 13) & 8u);
    const uint32_t q0 = ((uint32_t)__builtin_popcount(a0 & kLsbMask) + b0) & 1u;
    const uint32_t q1 = ((uint32_t)__builtin_popcount(a1 & kLsbMask) + b1) & 1u;
    p[6] = kc | ((b0 & 31u) << 1) | ((b1 & 31u) << 17);
    p[7] = kc | (((h0 << 1) | q0) << 1) | (((h1 << 1) | q1) << 17);
}

// int16 lattice values 2c -> fp16 pair of the coordinates c (exact)
__device__ __forceinline__ uint32_t pair_from_i16(int a, int b) {
    const h2_t r = {(_Float16)((float)a * 0.5f), (_Float16)((float)b * 0.5f)};
    return __builtin_bit_cast(uint32_t, r);
}

// fp16 pairs of coordinates c times the packed fp16 scales m = (s_lo, s_hi):
// fp16(c * s), one rounding of the exact product
template <int N>
__device__ __forceinline__ void mul_pairs(uint32_t p[N], uint32_t m) {
#pragma unroll
    for (int i = 0; i < N; i++)
        p[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, p[i]) * __builtin_bit_cast(h2_t, m));
}

__device__ __forceinline__ h8_t as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint4 u = make_uint4(a, b, c, d);
    return __builtin_bit_cast(h8_t, u);
}

// exception entry idx -> 8 lattice values 2c
__device__ __forceinline__ void exc_load(const int16_t* exc, int64_t idx, int v[8]) {
    const uint4 w = reinterpret_cast<const uint4*>(exc)[idx];
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = (int)(int16_t)(ww[i] & 0xffffu);
        v[2 * i + 1] = (int)(int16_t)(ww[i] >> 16);
    }
}

}  // namespace lq
