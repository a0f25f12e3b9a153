// dropout.cuh - the counter-based dropout mask, shared by dropout.cu and group_norm.cu.
//
// Generator: Philox-4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", 2011) with 7 rounds, the smallest count the paper found to pass BigCrush. One
// block gives four words = eight halfwords, one for each of eight draws. A draw is a 32-bit
// number u = (h << 16) | l with h from the block of half 0 and l from the block of half 1,
// kept when u >= T, T = rint(p 2^32). l decides only where h equals T >> 16 (one draw in
// 65536), so the second block is computed only by threads that meet such a draw: the mask
// has 32-bit resolution at the cost of 16 bits a draw.
#pragma once

#include "common.cuh"

namespace bsx {

constexpr int kRounds = 7;

// Launch arguments of a dropout mask.
struct DropArgs {
    uint32_t k0[kRounds], k1[kRounds];  // round keys: seed + r * Weyl constants, so that rounds read constants
    uint32_t step;                      // used when d_step is null
    const uint32_t* d_step;             // step read when the kernel runs
    uint32_t t_hi, t_lo;                // T = (t_hi << 16) + t_lo; T = 2^32 is 65535, 65536
    float scale;                        // 1 / (1 - p); 0 for p = 1
};

__device__ __forceinline__ uint4 philox7(const DropArgs& d, uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ d.k0[r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ d.k1[r];
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t drop_step(const DropArgs& d) { return d.d_step ? __ldg(d.d_step) : d.step; }

__device__ __forceinline__ uint32_t halfword(const uint4& w, int j) {
    const uint32_t v = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
    return j & 1 ? v >> 16 : v & 0xffffu;
}

__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Whether one of the eight halfwords equals t_hi, that is, whether some draw is decided by its
// low halfword: x - 0x00010001 borrows into a halfword's top bit where it was zero.
__device__ __forceinline__ bool any_tie(const DropArgs& d, const uint4& w) {
    const uint32_t t = d.t_hi | d.t_hi << 16;
    const uint32_t x = min_u16x2(min_u16x2(w.x ^ t, w.y ^ t), min_u16x2(w.z ^ t, w.w ^ t));
    return ((x - 0x00010001u) & ~x & 0x80008000u) != 0u;
}

// The kept draws of a block with ties.
__device__ __forceinline__ uint32_t tie_bits(const DropArgs& d, uint32_t step, uint32_t q0, uint32_t q1, const uint4& w) {
    const uint4 l = philox7(d, q0, q1, step, 1u);
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        keep |= (uint32_t)(halfword(w, j) > d.t_hi || (halfword(w, j) == d.t_hi && halfword(l, j) >= d.t_lo)) << j;
    return keep;
}

// Bit j: draw 8 q + j is kept.
__device__ __forceinline__ uint32_t keep8(const DropArgs& d, uint32_t step, uint64_t q) {
    const uint32_t q0 = (uint32_t)q, q1 = (uint32_t)(q >> 32);
    const uint4 w = philox7(d, q0, q1, step, 0u);
    if (any_tie(d, w)) return tie_bits(d, step, q0, q1, w);
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) keep |= (uint32_t)(halfword(w, j) > d.t_hi) << j;
    return keep;
}

// Draw m alone.
__device__ __forceinline__ bool keep1(const DropArgs& d, uint32_t step, uint64_t m) {
    const uint32_t q0 = (uint32_t)(m >> 3), q1 = (uint32_t)(m >> 35), j = (uint32_t)m & 7u;
    const uint4 w = philox7(d, q0, q1, step, 0u);
    const uint32_t a = j & 2 ? w.y : w.x, b = j & 2 ? w.w : w.z, h = (j & 4 ? b : a) >> (j & 1 ? 16 : 0) & 0xffffu;
    if (h != d.t_hi) return h > d.t_hi;
    const uint4 l = philox7(d, q0, q1, step, 1u);
    const uint32_t c = j & 2 ? l.y : l.x, e = j & 2 ? l.w : l.z;
    return ((j & 4 ? e : c) >> (j & 1 ? 16 : 0) & 0xffffu) >= d.t_lo;
}

// v[j] = draw 8 q + j kept ? v[j] scale : 0. Without a tie a draw is decided by one comparison on the
// whole word (odd draws) or on the word shifted up (even ones).
template <int V>
__device__ __forceinline__ void drop_values(const DropArgs& d, uint32_t step, uint64_t q, float (&v)[V]) {
    const uint32_t q0 = (uint32_t)q, q1 = (uint32_t)(q >> 32);
    const uint4 w = philox7(d, q0, q1, step, 0u);
    if (any_tie(d, w)) {
        const uint32_t keep = tie_bits(d, step, q0, q1, w);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = keep >> j & 1u ? v[j] * d.scale : 0.0f;
    } else {
        const uint32_t top = d.t_hi << 16 | 0xffffu;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t word = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
            v[j] = (j & 1 ? word : word << 16) > top ? v[j] * d.scale : 0.0f;
        }
    }
}

// Host: checks a configuration and fills the launch arguments. share is left to the caller.
const char* drop_args(const bsx_dropout_cfg* cfg, DropArgs* out);

}  // namespace bsx
