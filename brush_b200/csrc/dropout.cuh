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

// Launch arguments of a dropout mask.
struct DropArgs {
    uint32_t k0, k1;          // seed
    uint32_t step;            // used when d_step is null
    const uint32_t* d_step;   // step read when the kernel runs
    uint32_t t_hi, t_lo;      // T >> 16 (0..65536) and T & 0xffff
    float scale;              // 1 / (1 - p); 0 for p = 1
};

__device__ __forceinline__ uint4 philox7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t drop_step(const DropArgs& d) { return d.d_step ? __ldg(d.d_step) : d.step; }

// Bit j: draw 8 q + j is kept.
__device__ __forceinline__ uint32_t keep8(const DropArgs& d, uint32_t step, uint64_t q) {
    const uint32_t q0 = (uint32_t)q, q1 = (uint32_t)(q >> 32);
    const uint4 hw = philox7(q0, q1, step, 0u, d.k0, d.k1);
    const uint32_t h[4] = {hw.x, hw.y, hw.z, hw.w};
    uint32_t keep = 0, tie = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t v = (j & 1) ? h[j >> 1] >> 16 : h[j >> 1] & 0xffffu;
        keep |= (uint32_t)(v > d.t_hi) << j;
        tie |= (uint32_t)(v == d.t_hi) << j;
    }
    if (tie) {
        const uint4 lw = philox7(q0, q1, step, 1u, d.k0, d.k1);
        const uint32_t l[4] = {lw.x, lw.y, lw.z, lw.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t v = (j & 1) ? l[j >> 1] >> 16 : l[j >> 1] & 0xffffu;
            keep |= (uint32_t)(v >= d.t_lo && (tie >> j & 1u)) << j;
        }
    }
    return keep;
}

// Host: checks a configuration and fills the launch arguments. share is left to the caller.
const char* drop_args(const bsx_dropout_cfg* cfg, DropArgs* out);

}  // namespace bsx
