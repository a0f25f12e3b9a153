// group_norm.cuh - what the group-norm kernels share: arguments, the cut of a tensor into
// blocks, per-thread statistics, sums over groups inside a block, and the activation.
//
// Layout. A sample is a run of pixels C elements long. Threads read vectors of V elements; a
// "row" is the shortest run that starts and ends on a pixel and on a vector: C / gcd(C, V)
// vectors, lcm(C, V) elements. A block takes k rows at a time with one vector a thread, so a
// thread meets the same V channels in every row: their weights, biases and statistics stay in
// its registers, odd channel counts included. Wide rows are cut into tiles of columns.
#pragma once

#include "dropout.cuh"
#include "elem.cuh"

namespace bsx {
namespace norm {

constexpr int kThreads = 512;     // most threads of a block
constexpr int kBatch = 8;         // vectors of a thread in the kernels for small samples
constexpr int kFlight = 4;        // vectors of a thread in flight in the kernels for large samples
constexpr int kBatchBwd = 4;      // the same two for the backward, of x and of v each
constexpr int kFlightBwd = 2;
constexpr uint32_t kMaxBlocks = 512;  // most blocks of a kernel for large samples

struct Args {
    const void* x;
    const void* v;       // backward: gradient of the output
    const void* weight;  // null: 1
    const void* bias;    // null: 0
    void* out;           // forward: out, backward: v_x
    float* mean;
    float* rstd;
    float* ws;
    void* v_weight;
    void* v_bias;
    uint64_t n, pixels;
    uint32_t c, groups, per;  // per = c / groups
    float eps;
    int param_f32;
    DropArgs drop;
};

// How the tensor is cut (plan_for in group_norm.cu).
struct Plan {
    uint64_t vecs;       // vectors of a sample
    uint64_t rows;       // rows of a sample; the last may be cut short
    uint64_t per_block;  // large samples: rows of a block, over tiles and samples in order
    uint32_t rv;         // vectors of a row
    uint32_t cols;       // vectors of a tile's row; the last tile may have fewer
    uint32_t tiles;
    uint32_t k;          // rows a block takes at a time
    uint32_t gl;         // most groups of a tile
    uint32_t keep;       // large samples: iterations whose vectors stay in shared memory
    uint32_t threads, blocks;
    uint32_t v;          // elements of a vector
    int small;           // one block per (sample, tile), everything in registers
};

template <class T>
__device__ __forceinline__ float param(const void* p, int f32, uint32_t c, float without) {
    if (!p) return without;
    return f32 ? __ldg((const float*)p + c) : to_f(((const T*)p)[c]);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// act(z) = z s(w(z)), s the logistic function: w = z (silu), or 2 sqrt(2/pi) (z + 0.044715 z^3)
// (gelu in its tanh form, because (1 + tanh(t)) / 2 = s(2 t)). s = 1 / (1 + 2^(-w log2 e)), with
// the approximate exponential and reciprocal (2 and 1 ulp); both ends are right: the exponential
// overflows to infinity and s to 0, or vanishes and s is 1.
constexpr float kLog2e = 1.4426950408889634f, kGelu1 = 1.5957691216057308f, kGelu3 = 0.044715f;
template <int ACT>
__device__ __forceinline__ float gate(float z) {
    if (ACT == BSX_ACT_NONE) return 1.0f;
    float e;
    if (ACT == BSX_ACT_SILU) e = z * -kLog2e;
    else e = z * __fmaf_rn(z * z, -kLog2e * kGelu1 * kGelu3, -kLog2e * kGelu1);
    return rcp_fast(1.0f + exp2_fast(e));
}
template <int ACT>
__device__ __forceinline__ float act(float z) {
    return ACT == BSX_ACT_NONE ? z : z * gate<ACT>(z);
}
// act'(z) = s + z s (1 - s) w'(z)
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if (ACT == BSX_ACT_NONE) return 1.0f;
    const float s = gate<ACT>(z);
    float dw = z;
    if (ACT == BSX_ACT_GELU_TANH) dw = z * __fmaf_rn(z * z, 3.0f * kGelu1 * kGelu3, kGelu1);
    return __fmaf_rn(__fmaf_rn(-s, s, s), dw, s);
}

// The columns and groups of a tile. Items are vectors where a vector lies in one group (L = 1), else elements.
struct Tile {
    uint32_t cols;         // vectors in the tile's row
    uint32_t c0, c1;       // channels
    uint32_t g0, groups;   // groups that have channels here
    uint32_t stride;       // items from a channel to its next copy in the block
    uint32_t copies;       // copies of the channels in the block's k rows
};
template <int V, int L>
__device__ __forceinline__ Tile tile_of(const Args& a, const Plan& p, uint32_t t) {
    Tile r;
    r.cols = min(p.cols, p.rv - t * p.cols);
    if (p.tiles == 1) r.c0 = 0, r.c1 = a.c;
    else r.c0 = t * p.cols * V, r.c1 = r.c0 + r.cols * V;
    r.g0 = r.c0 / a.per;
    r.groups = (r.c1 - 1) / a.per - r.g0 + 1;
    r.stride = (r.c1 - r.c0) / (V / L);
    r.copies = p.k * r.cols * L / r.stride;
    return r;
}

// Sums over the tile's groups of one value per item (thread t holds items t L ... t L + L - 1 of the block's
// k rows), in a fixed order: a warp, or several where groups are few, walks each group's items. After the
// call sum[g] holds group g0 + g for all threads. Starts and ends with a barrier.
template <int V, int L, bool PAIR>
__device__ __forceinline__ void group_sums(const Args& a, const Tile& t, const float (&x)[L], const float (&y)[L],
                                           bool active, float* part, float* warp_sum, float2* sum) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const uint32_t half = blockDim.x * L;  // the pair's second values
    __syncthreads();
#pragma unroll
    for (int j = 0; j < L; ++j) {
        part[tid * L + j] = active ? x[j] : 0.0f;
        if (PAIR) part[half + tid * L + j] = active ? y[j] : 0.0f;
    }
    __syncthreads();
    const uint32_t share = max(1u, warps / t.groups);  // warps of a group
    for (uint32_t u = warp; u < t.groups * share; u += warps) {
        const uint32_t g = u / share, q = u - g * share;
        const uint32_t lo = (max((t.g0 + g) * a.per, t.c0) - t.c0) / (V / L);
        const uint32_t hi = (min((t.g0 + g + 1) * a.per, t.c1) - t.c0) / (V / L);
        const uint32_t width = hi - lo, count = t.copies * width;
        const float inv = 1.0f / (float)width;
        float s = 0.0f, s2 = 0.0f;
        for (uint32_t i = q * 32 + lane; i < count; i += 32 * share) {
            const uint32_t m = (uint32_t)(((float)i + 0.5f) * inv);  // i / width: i < 2^13, far from a whole number
            const uint32_t at = m * t.stride + lo + (i - m * width);
            s += part[at];
            if (PAIR) s2 += part[half + at];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            s += __shfl_xor_sync(~0u, s, o);
            if (PAIR) s2 += __shfl_xor_sync(~0u, s2, o);
        }
        if (lane == 0) {
            warp_sum[u * 2] = s;
            warp_sum[u * 2 + 1] = s2;
        }
    }
    __syncthreads();
    for (uint32_t g = tid; g < t.groups; g += blockDim.x) {
        float s = 0.0f, s2 = 0.0f;
        for (uint32_t q = 0; q < share; ++q) {
            s += warp_sum[(g * share + q) * 2];
            s2 += warp_sum[(g * share + q) * 2 + 1];
        }
        sum[g] = make_float2(s, s2);
    }
    __syncthreads();
}

// Floats of shared memory that group_sums takes: part, warp_sum, sum.
inline uint32_t sums_floats(uint32_t threads, uint32_t lanes, uint32_t gl, bool pair) {
    return threads * lanes * (pair ? 2 : 1) + 2 * (gl > kThreads / 32 ? gl : kThreads / 32) + 2 * gl;
}
template <int L, bool PAIR>
struct Scratch {
    float *part, *warp_sum;
    float2* sum;
    float* end;
    __device__ __forceinline__ Scratch(float* smem, uint32_t gl) {
        part = smem;
        warp_sum = part + blockDim.x * L * (PAIR ? 2 : 1);
        sum = (float2*)(warp_sum + 2 * max(gl, (uint32_t)kThreads / 32));
        end = (float*)(sum + gl);
    }
};

// Group of lane j of a vector that starts at channel c, relative to the tile's first.
template <int V, int L>
__device__ __forceinline__ uint32_t group_at(const Args& a, const Tile& t, uint32_t c, int j) {
    uint32_t ch = c + j;
    if (L > 1) while (ch >= a.c) ch -= a.c;  // rows of several pixels
    return ch / a.per - t.g0;
}
__device__ __forceinline__ uint32_t channel_at(const Args& a, uint32_t c, int j) {
    uint32_t ch = c + j;
    while (ch >= a.c) ch -= a.c;
    return ch;
}

// drop for V elements from flat element `at` (V divides it, and 8).
template <int V>
__device__ __forceinline__ void drop_vector(const DropArgs& d, uint32_t step, uint64_t at, float (&v)[V]) {
    if constexpr (V == 8) {
        drop_values<8>(d, step, at >> 3, v);
    } else {
        const uint32_t keep = keep8(d, step, at >> 3) >> (at & 7);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = keep >> j & 1u ? v[j] * d.scale : 0.0f;
    }
}

// A block's share of one (tile, sample) of a large tensor.
struct Segment {
    uint64_t n, r0, at;   // sample, first row, first element of the thread's first vector
    uint32_t tile, c;     // tile, channel of the thread's first element
    uint32_t iters, cnt;  // iterations of the block, of this thread
    uint32_t pixels;      // float-exact below 2^24; counts enter as float
};
__device__ __forceinline__ uint32_t segment_iters(const Plan& p, uint64_t len) { return (uint32_t)((len + p.k - 1) / p.k); }

template <int V, int L>
__device__ __forceinline__ Segment segment_of(const Args& a, const Plan& p, uint64_t u, uint64_t from, uint64_t to,
                                              Tile& t) {
    Segment s;
    s.tile = (uint32_t)(u / a.n);
    s.n = u - s.tile * a.n;
    s.r0 = from - u * p.rows;
    t = tile_of<V, L>(a, p, s.tile);
    const uint64_t r1 = to - u * p.rows;
    const uint32_t tid = threadIdx.x, row = tid / t.cols, col = s.tile * p.cols + tid - row * t.cols;
    const uint64_t lim = r1 - (r1 == p.rows && (p.rows - 1) * p.rv + col >= p.vecs);  // rows of this column
    s.iters = segment_iters(p, r1 - s.r0);
    s.cnt = row < p.k && s.r0 + row < lim ? (uint32_t)((lim - s.r0 - row + p.k - 1) / p.k) : 0;
    s.at = (s.n * p.vecs + (s.r0 + row) * p.rv + col) * V;
    s.c = col * V % a.c;
    const uint64_t e1 = r1 * p.rv * V;
    s.pixels = (uint32_t)(((e1 < p.vecs * V ? e1 : p.vecs * V) - s.r0 * p.rv * V) / a.c);
    return s;
}

// Iterations of block b's run, over its segments.
__device__ __forceinline__ uint32_t run_iters(const Plan& p, uint64_t w0, uint64_t w1) {
    uint32_t all = 0;
    for (uint64_t w = w0; w < w1;) {
        const uint64_t next = (w / p.rows + 1) * p.rows, to = next < w1 ? next : w1;
        all += segment_iters(p, to - w);
        w = to;
    }
    return all;
}

// Host side, one per element type (group_norm_{f32,bf16,f16}.cu). `whole`: a vector lies in one group.
struct Call {
    const Args* a;
    Plan* p;
    int act;
    bool drop, whole, bwd;
    int device;
    cudaStream_t stream;
};
template <class T>
cudaError_t launch(const Call& c);

}  // namespace norm
}  // namespace bsx
