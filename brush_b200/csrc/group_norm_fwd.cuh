// group_norm_fwd.cuh - the forward kernels of group norm.
#pragma once

#include <cooperative_groups.h>

#include "group_norm.cuh"

namespace bsx {
namespace norm {

// A thread's place in a tile and what it needs of its V channels.
template <class T, int V, int L>
struct Lanes {
    float a[V], b[V], mean[L];

    __device__ __forceinline__ void params(const Args& g, uint32_t c) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t ch = channel_at(g, c, j);
            a[j] = param<T>(g.weight, g.param_f32, ch, 1.0f);
            b[j] = param<T>(g.bias, g.param_f32, ch, 0.0f);
        }
    }
    // stat[g]: mean and rstd
    __device__ __forceinline__ void fold(const Args& g, const Tile& t, uint32_t c, const float2* stat) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j < L || L > 1) {
                const float2 s = stat[group_at<V, L>(g, t, c, j)];
                mean[j] = s.x;
                a[j] *= s.y;
            } else {
                a[j] *= stat[group_at<V, L>(g, t, c, 0)].y;
            }
        }
    }
    template <int ACT>
    __device__ __forceinline__ void apply(float (&v)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = act<ACT>(__fmaf_rn(v[j] - mean[L > 1 ? j : 0], a[j], b[j]));
    }
};

// Small samples: one block per (sample, tile), at most kBatch vectors a thread, held in registers between
// the sums and the result: x is read once. Mean, then the squares of the deviations from it.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) small_fwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    const Scratch<L, false> s(smem, p.gl);
    const uint32_t tid = threadIdx.x, tile = blockIdx.x % p.tiles;
    const uint64_t n = blockIdx.x / p.tiles;
    const Tile t = tile_of<V, L>(a, p, tile);
    const uint32_t row = tid / t.cols, col = tile * p.cols + tid - row * t.cols;
    const bool active = row < p.k;
    const uint32_t rows = (uint32_t)p.rows - ((p.rows - 1) * p.rv + col >= p.vecs);  // of this column
    const uint32_t cnt = active && row < rows ? (rows - row + p.k - 1) / p.k : 0;
    const uint64_t at = (n * p.vecs + (uint64_t)row * p.rv + col) * V;
    const uint32_t step = p.k * p.rv * V;
    const T* x = (const T*)a.x + at;
    Pack<T, V> raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) raw[i].load(x + (uint64_t)i * step);
    const uint32_t c = col * V % a.c;
    Lanes<T, V, L> lanes;
    if (active) lanes.params(a, c);

    const float m = (float)(p.vecs * V / a.groups);  // values of a group
    float sum[L] = {};
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[L > 1 ? j : 0] += f[j];
        }
    group_sums<V, L, false>(a, t, sum, sum, active, s.part, s.warp_sum, s.sum);
    float mean[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
        mean[j] = active ? s.sum[group_at<V, L>(a, t, c, j)].x / m : 0.0f;
        sum[j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = f[j] - mean[L > 1 ? j : 0];
                sum[L > 1 ? j : 0] = __fmaf_rn(d, d, sum[L > 1 ? j : 0]);
            }
        }
    float* means = s.end;  // [gl]: s.sum is filled again
    for (uint32_t g = tid; g < t.groups; g += blockDim.x) means[g] = s.sum[g].x / m;
    group_sums<V, L, false>(a, t, sum, sum, active, s.part, s.warp_sum, s.sum);
    for (uint32_t g = tid; g < t.groups; g += blockDim.x) {
        const float rstd = 1.0f / sqrtf(s.sum[g].x / m + a.eps);
        s.sum[g] = make_float2(means[g], rstd);
        a.mean[n * a.groups + t.g0 + g] = means[g];
        a.rstd[n * a.groups + t.g0 + g] = rstd;
    }
    __syncthreads();
    if (cnt == 0) return;
    lanes.fold(a, t, c, s.sum);
    const uint32_t dstep = DROP ? drop_step(a.drop) : 0u;
    T* out = (T*)a.out + at;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
            lanes.template apply<ACT>(f);
            if (DROP) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, f);
            raw[i].set(f);
            raw[i].store(out + (uint64_t)i * step);
        }
}

// Large samples: one cooperative launch. The rows of all samples, tile after tile, are dealt to the blocks in
// runs of per_block. First pass: mean and sum of squared deviations of each group in each run (from a pivot,
// the mean of a thread's first vectors, so that no large mean cancels), to the workspace. Grid barrier. Second
// pass, last row first: the runs' statistics are joined, and the rows are normalised from shared memory where
// the first pass left its last `keep` iterations, and else from where they are nearest, L2 if they were read late.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads, 1) large_fwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    const Scratch<L, false> s(smem, p.gl);
    Pack<T, V>* kept = (Pack<T, V>*)(((uintptr_t)s.end + 15) & ~(uintptr_t)15);  // [keep][threads]
    const uint32_t tid = threadIdx.x, step = p.k * p.rv * V;
    const uint64_t total = p.rows * a.n * p.tiles, w0 = blockIdx.x * p.per_block;
    const uint64_t w1 = w0 + p.per_block < total ? w0 + p.per_block : total;
    const uint32_t all = run_iters(p, w0, w1);
    const uint32_t kept_from = all > p.keep ? all - p.keep : 0;
    float4* slots = (float4*)a.ws;  // [(block + unit) gl + group]: mean, squared deviations, count

    uint32_t it = 0;
    for (uint64_t w = w0; w < w1;) {
        const uint64_t u = w / p.rows, to = (u + 1) * p.rows < w1 ? (u + 1) * p.rows : w1;
        Tile t;
        const Segment g = segment_of<V, L>(a, p, u, w, to, t);
        const T* x = (const T*)a.x + g.at;
        float pivot[L] = {}, sum[L] = {}, sq[L] = {};
        Pack<T, V> cur[kFlight], nxt[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i)
            if (i < g.cnt) cur[i].load(x + (uint64_t)i * step);
        for (uint32_t i0 = 0; i0 < g.iters; i0 += kFlight) {
#pragma unroll
            for (int i = 0; i < kFlight; ++i)
                if (i0 + kFlight + i < g.cnt) nxt[i].load(x + (uint64_t)(i0 + kFlight + i) * step);
            if (i0 == 0 && g.cnt) {
                const uint32_t have = g.cnt < kFlight ? g.cnt : kFlight;
#pragma unroll
                for (int i = 0; i < kFlight; ++i)
                    if (i < have) {
                        float f[V];
                        cur[i].get(f);
#pragma unroll
                        for (int j = 0; j < V; ++j) pivot[L > 1 ? j : 0] += f[j];
                    }
                const float inv = 1.0f / (float)(have * (V / L));
#pragma unroll
                for (int j = 0; j < L; ++j) pivot[j] *= inv;
            }
#pragma unroll
            for (int i = 0; i < kFlight; ++i)
                if (i0 + i < g.cnt) {
                    float f[V];
                    cur[i].get(f);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int l = L > 1 ? j : 0;
                        const float d = f[j] - pivot[l];
                        sum[l] += d;
                        sq[l] = __fmaf_rn(d, d, sq[l]);
                    }
                    if (it + i0 + i >= kept_from) kept[(it + i0 + i - kept_from) * blockDim.x + tid] = cur[i];
                }
#pragma unroll
            for (int i = 0; i < kFlight; ++i) cur[i] = nxt[i];
        }
        const float cnt = (float)g.cnt * (V / L);
        float mean[L], dev[L], val[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float d = g.cnt ? sum[j] / cnt : 0.0f;
            mean[j] = pivot[j] + d;
            dev[j] = __fmaf_rn(-sum[j], d, sq[j]);
            if (dev[j] < 0.0f) dev[j] = 0.0f;
            val[j] = cnt * mean[j];
        }
        group_sums<V, L, false>(a, t, val, val, g.cnt != 0, s.part, s.warp_sum, s.sum);
        float gm[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            gm[j] = 0.0f;
            if (g.cnt) {
                const uint32_t q = group_at<V, L>(a, t, g.c, j);
                const uint32_t width = min((t.g0 + q + 1) * a.per, t.c1) - max((t.g0 + q) * a.per, t.c0);
                gm[j] = s.sum[q].x / ((float)g.pixels * (float)width);
            }
            const float d = mean[j] - gm[j];
            val[j] = __fmaf_rn(cnt * d, d, dev[j]);
        }
        float4* slot = slots + (blockIdx.x + u) * p.gl;
        for (uint32_t q = tid; q < t.groups; q += blockDim.x) {
            const uint32_t width = min((t.g0 + q + 1) * a.per, t.c1) - max((t.g0 + q) * a.per, t.c0);
            const float count = (float)g.pixels * (float)width;
            slot[q] = make_float4(s.sum[q].x / count, 0.0f, count, 0.0f);
        }
        group_sums<V, L, false>(a, t, val, val, g.cnt != 0, s.part, s.warp_sum, s.sum);
        for (uint32_t q = tid; q < t.groups; q += blockDim.x) slot[q].y = s.sum[q].x;
        it += g.iters;
        w = to;
    }

    cooperative_groups::this_grid().sync();

    const uint32_t dstep = DROP ? drop_step(a.drop) : 0u;
    const uint32_t lane = tid & 31, warp = tid >> 5;
    for (uint64_t end = w1; end > w0;) {
        const uint64_t u = (end - 1) / p.rows, from = u * p.rows > w0 ? u * p.rows : w0;
        Tile t;
        const Segment g = segment_of<V, L>(a, p, u, from, end, t);
        Lanes<T, V, L> lanes;
        if (g.cnt) lanes.params(a, g.c);
        __syncthreads();  // s.sum of the segment before is read no more
        for (uint32_t q = warp; q < t.groups; q += blockDim.x / 32) {
            const uint32_t grp = t.g0 + q;
            const uint32_t tile_c = p.tiles == 1 ? a.c : p.cols * V;
            const uint32_t t0 = grp * a.per / tile_c, t1 = ((grp + 1) * a.per - 1) / tile_c;
            float sum = 0.0f, count = 0.0f;
            for (uint32_t k = t0; k <= t1; ++k) {
                const uint64_t uu = k * a.n + g.n;
                const uint64_t b0 = uu * p.rows / p.per_block, b1 = ((uu + 1) * p.rows - 1) / p.per_block;
                const uint32_t at = grp - k * tile_c / a.per;
                for (uint64_t b = b0 + lane; b <= b1; b += 32) {
                    const float4 v = __ldcg(slots + (b + uu) * p.gl + at);
                    sum = __fmaf_rn(v.x, v.z, sum);
                    count += v.z;
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sum += __shfl_xor_sync(~0u, sum, o);
                count += __shfl_xor_sync(~0u, count, o);
            }
            const float mean = sum / count;
            float dev = 0.0f;
            for (uint32_t k = t0; k <= t1; ++k) {
                const uint64_t uu = k * a.n + g.n;
                const uint64_t b0 = uu * p.rows / p.per_block, b1 = ((uu + 1) * p.rows - 1) / p.per_block;
                const uint32_t at = grp - k * tile_c / a.per;
                for (uint64_t b = b0 + lane; b <= b1; b += 32) {
                    const float4 v = __ldcg(slots + (b + uu) * p.gl + at);
                    const float d = v.x - mean;
                    dev += __fmaf_rn(v.z * d, d, v.y);
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) dev += __shfl_xor_sync(~0u, dev, o);
            const float rstd = 1.0f / sqrtf(dev / count + a.eps);
            if (lane == 0) {
                s.sum[q] = make_float2(mean, rstd);
                if (g.r0 == 0 && grp * a.per >= t.c0) {
                    a.mean[g.n * a.groups + grp] = mean;
                    a.rstd[g.n * a.groups + grp] = rstd;
                }
            }
        }
        __syncthreads();
        it -= g.iters;
        if (g.cnt) {
            lanes.fold(a, t, g.c, s.sum);
            const T* x = (const T*)a.x + g.at;
            T* out = (T*)a.out + g.at;
            for (uint32_t i1 = (g.cnt + kFlight - 1) / kFlight * kFlight; i1 > 0; i1 -= kFlight) {
                Pack<T, V> raw[kFlight];
#pragma unroll
                for (int i = kFlight - 1; i >= 0; --i) {
                    const uint32_t k = i1 - kFlight + i;
                    if (k < g.cnt) {
                        if (it + k >= kept_from) raw[i] = kept[(it + k - kept_from) * blockDim.x + tid];
                        else raw[i].load(x + (uint64_t)k * step);
                    }
                }
#pragma unroll
                for (int i = kFlight - 1; i >= 0; --i) {
                    const uint32_t k = i1 - kFlight + i;
                    if (k < g.cnt) {
                        float f[V];
                        raw[i].get(f);
                        lanes.template apply<ACT>(f);
                        if (DROP) drop_vector<V>(a.drop, dstep, g.at + (uint64_t)k * step, f);
                        raw[i].set(f);
                        raw[i].store(out + (uint64_t)k * step);
                    }
                }
            }
        }
        end = from;
    }
}

}  // namespace norm
}  // namespace bsx
