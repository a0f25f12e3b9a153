// group_norm_bwd.cuh - the backward kernels of group norm.
#pragma once

#include <cooperative_groups.h>

#include "group_norm.cuh"

namespace bsx {
namespace norm {

// What a thread needs of its V channels.
template <class T, int V, int L>
struct GradLanes {
    float w[V], b[V], mean[L], rstd[L];

    __device__ __forceinline__ void params(const Args& a, uint32_t c) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t ch = channel_at(a, c, j);
            w[j] = param<T>(a.weight, a.param_f32, ch, 1.0f);
            b[j] = param<T>(a.bias, a.param_f32, ch, 0.0f);
        }
    }
    __device__ __forceinline__ void stats(const Args& a, uint64_t n, uint32_t c) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const uint64_t at = n * a.groups + channel_at(a, c, j) / a.per;
            mean[j] = __ldg(a.mean + at);
            rstd[j] = __ldg(a.rstd + at);
        }
    }
    // x becomes xh, v becomes dz
    template <int ACT>
    __device__ __forceinline__ void grads(float (&x)[V], float (&v)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x[j] = (x[j] - mean[L > 1 ? j : 0]) * rstd[L > 1 ? j : 0];
            if (ACT != BSX_ACT_NONE) v[j] *= act_grad<ACT>(__fmaf_rn(x[j], w[j], b[j]));
        }
    }
};

// s1 and s2 of a thread's groups, divided by the values of a group and multiplied by rstd.
template <class T, int V, int L>
struct GroupGrad {
    float s1[L], s2[L];
    __device__ __forceinline__ void take(const Args& a, const Tile& t, uint32_t c, const float2* sum, float m,
                                         const float (&rstd)[L]) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float2 s = sum[group_at<V, L>(a, t, c, j)];
            s1[j] = s.x / m * rstd[j];
            s2[j] = s.y / m * rstd[j];
        }
    }
    __device__ __forceinline__ void apply(const GradLanes<T, V, L>& g, const float (&xh)[V], const float (&dz)[V],
                                          float (&out)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int l = L > 1 ? j : 0;
            out[j] = __fmaf_rn(g.w[j] * g.rstd[l], dz[j], -__fmaf_rn(xh[j], s2[l], s1[l]));
        }
    }
};

// A block's sums over its copies of each channel of a tile, to two arrays `to`: [channel - c0].
template <int V>
__device__ __forceinline__ void channel_sums(const Tile& t, uint32_t k, const float (&x)[V], const float (&y)[V],
                                             bool active, float* part, float2* to) {
    const uint32_t tid = threadIdx.x, half = blockDim.x * V;
    const uint32_t width = t.c1 - t.c0, copies = k * t.cols * V / width;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        part[tid * V + j] = active ? x[j] : 0.0f;
        part[half + tid * V + j] = active ? y[j] : 0.0f;
    }
    __syncthreads();
    // q threads a channel sum every q-th copy into the first q copies, then one adds those
    uint32_t q = blockDim.x / width;
    if (q > copies) q = copies;
    if (q > 1) {
        const uint32_t z = tid / width, i = tid - z * width;
        if (z < q) {
            float s = 0.0f, s2 = 0.0f;
            for (uint32_t m = z; m < copies; m += q) {
                s += part[m * width + i];
                s2 += part[half + m * width + i];
            }
            part[z * width + i] = s;
            part[half + z * width + i] = s2;
        }
        __syncthreads();
    } else {
        q = copies;
    }
    for (uint32_t i = tid; i < width; i += blockDim.x) {
        float s = 0.0f, s2 = 0.0f;
        for (uint32_t m = 0; m < q; ++m) {
            s += part[m * width + i];
            s2 += part[half + m * width + i];
        }
        to[i] = make_float2(s, s2);
    }
    __syncthreads();
}

// Parameter gradients of one channel from its partial sums (x: bias, y: weight), by a warp.
template <class T>
__device__ __forceinline__ void join_channel(const Args& a, uint32_t c, const float2* from, uint64_t count,
                                             uint64_t stride) {
    float s = 0.0f, s2 = 0.0f;
    for (uint64_t i = threadIdx.x & 31; i < count; i += 32) {
        const float2 v = __ldcg(from + i * stride);
        s += v.x;
        s2 += v.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(~0u, s, o);
        s2 += __shfl_xor_sync(~0u, s2, o);
    }
    if ((threadIdx.x & 31) == 0) {
        if (a.v_bias) {
            if (a.param_f32) ((float*)a.v_bias)[c] = s;
            else ((T*)a.v_bias)[c] = from_f<T>(s);
        }
        if (a.v_weight) {
            if (a.param_f32) ((float*)a.v_weight)[c] = s2;
            else ((T*)a.v_weight)[c] = from_f<T>(s2);
        }
    }
}

// Small samples: a block takes (sample, tile) pairs of one tile, x and v in registers between the sums and the
// result. Channel sums go on over its samples and to the workspace at the end, [block of the tile][channel];
// after a grid barrier (cooperative launch) a warp a channel adds them up.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) small_bwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    const Scratch<V, true> s(smem, p.gl);  // V: channel_sums keeps single channels
    const uint32_t tid = threadIdx.x, tile = blockIdx.x % p.tiles;
    const Tile t = tile_of<V, L>(a, p, tile);
    const uint32_t row = tid / t.cols, col = tile * p.cols + tid - row * t.cols;
    const bool active = row < p.k;
    const uint32_t rows = (uint32_t)p.rows - ((p.rows - 1) * p.rv + col >= p.vecs);
    const uint32_t cnt = active && row < rows ? (rows - row + p.k - 1) / p.k : 0;
    const uint32_t step = p.k * p.rv * V, c = col * V % a.c;
    const uint32_t dstep = DROP ? drop_step(a.drop) : 0u;
    const float m = (float)(p.vecs * V / a.groups);
    GradLanes<T, V, L> lanes;
    if (active) lanes.params(a, c);
    float acc_a[V] = {}, acc_b[V] = {};
    for (uint64_t n = blockIdx.x / p.tiles; n < a.n; n += gridDim.x / p.tiles) {
        const uint64_t at = (n * p.vecs + (uint64_t)row * p.rv + col) * V;
        Pack<T, V> rx[kBatchBwd], rv[kBatchBwd];
#pragma unroll
        for (int i = 0; i < kBatchBwd; ++i)
            if (i < cnt) {
                rx[i].load((const T*)a.x + at + (uint64_t)i * step);
                rv[i].load((const T*)a.v + at + (uint64_t)i * step);
            }
        if (active) lanes.stats(a, n, c);
        float s1[L] = {}, s2[L] = {};
#pragma unroll
        for (int i = 0; i < kBatchBwd; ++i)
            if (i < cnt) {
                float x[V], v[V];
                rx[i].get(x);
                rv[i].get(v);
                if (DROP) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, v);
                lanes.template grads<ACT>(x, v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float b = v[j] * x[j];
                    acc_a[j] += v[j];
                    acc_b[j] += b;
                    s1[L > 1 ? j : 0] = __fmaf_rn(lanes.w[j], v[j], s1[L > 1 ? j : 0]);
                    s2[L > 1 ? j : 0] = __fmaf_rn(lanes.w[j], b, s2[L > 1 ? j : 0]);
                }
            }
        group_sums<V, L, true>(a, t, s1, s2, active, s.part, s.warp_sum, s.sum);
        if (cnt) {
            GroupGrad<T, V, L> gg;
            gg.take(a, t, c, s.sum, m, lanes.rstd);
#pragma unroll
            for (int i = 0; i < kBatchBwd; ++i)
                if (i < cnt) {
                    float x[V], v[V], o[V];
                    rx[i].get(x);
                    rv[i].get(v);
                    if (DROP) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, v);
                    lanes.template grads<ACT>(x, v);
                    gg.apply(lanes, x, v, o);
                    rx[i].set(o);
                    rx[i].store((T*)a.out + at + (uint64_t)i * step);
                }
        }
    }
    if (!a.v_weight && !a.v_bias) return;  // of all blocks alike
    float2* ws = (float2*)a.ws;
    channel_sums<V>(t, p.k, acc_a, acc_b, active, s.part, ws + (uint64_t)(blockIdx.x / p.tiles) * a.c + t.c0);
    cooperative_groups::this_grid().sync();
    for (uint32_t ch = blockIdx.x * (blockDim.x / 32) + tid / 32; ch < a.c; ch += gridDim.x * (blockDim.x / 32))
        join_channel<T>(a, ch, ws + ch, gridDim.x / p.tiles, a.c);
}

// Large samples: dealt like the forward's. First pass: sums of gamma dz and gamma dz xh of each group in each run,
// and of dz and dz xh of each channel in each block, to the workspace. Grid barrier. Second pass, last row first:
// the group sums are joined and v_x formed, from shared memory for the last `keep` iterations; the channels are
// dealt to the warps of the grid.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads, 1) large_bwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    const Scratch<V, true> s(smem, p.gl);
    Pack<T, V>* kept = (Pack<T, V>*)(((uintptr_t)s.end + 15) & ~(uintptr_t)15);  // [keep][x, v][threads]
    const uint32_t tid = threadIdx.x, step = p.k * p.rv * V;
    const uint64_t total = p.rows * a.n * p.tiles, w0 = blockIdx.x * p.per_block;
    const uint64_t w1 = w0 + p.per_block < total ? w0 + p.per_block : total;
    const uint32_t all = run_iters(p, w0, w1), kept_from = all > p.keep ? all - p.keep : 0;
    const uint32_t dstep = DROP ? drop_step(a.drop) : 0u;
    const uint32_t tile_c = p.tiles == 1 ? a.c : p.cols * V;  // channels of a full tile
    float2* slots = (float2*)a.ws;                             // [(block + unit) gl + group]
    float2* chans = slots + (gridDim.x + p.tiles * a.n) * p.gl;  // [(block + tile) tile_c + channel - c0]
    const bool params = a.v_weight || a.v_bias;

    uint32_t it = 0;
    float acc_a[V] = {}, acc_b[V] = {};
    for (uint64_t w = w0; w < w1;) {
        const uint64_t u = w / p.rows, to = (u + 1) * p.rows < w1 ? (u + 1) * p.rows : w1;
        Tile t;
        const Segment g = segment_of<V, L>(a, p, u, w, to, t);
        const T *x = (const T*)a.x + g.at, *v = (const T*)a.v + g.at;
        GradLanes<T, V, L> lanes;
        float sa[V] = {}, sb[V] = {};
        Pack<T, V> cx[kFlightBwd], cv[kFlightBwd], nx[kFlightBwd], nv[kFlightBwd];
#pragma unroll
        for (int i = 0; i < kFlightBwd; ++i)
            if (i < g.cnt) {
                cx[i].load(x + (uint64_t)i * step);
                cv[i].load(v + (uint64_t)i * step);
            }
        if (g.cnt) {
            lanes.params(a, g.c);
            lanes.stats(a, g.n, g.c);
        }
        for (uint32_t i0 = 0; i0 < g.iters; i0 += kFlightBwd) {
#pragma unroll
            for (int i = 0; i < kFlightBwd; ++i)
                if (i0 + kFlightBwd + i < g.cnt) {
                    nx[i].load(x + (uint64_t)(i0 + kFlightBwd + i) * step);
                    nv[i].load(v + (uint64_t)(i0 + kFlightBwd + i) * step);
                }
#pragma unroll
            for (int i = 0; i < kFlightBwd; ++i)
                if (i0 + i < g.cnt) {
                    float fx[V], fv[V];
                    cx[i].get(fx);
                    cv[i].get(fv);
                    if (DROP) drop_vector<V>(a.drop, dstep, g.at + (uint64_t)(i0 + i) * step, fv);
                    lanes.template grads<ACT>(fx, fv);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        sa[j] += fv[j];
                        sb[j] = __fmaf_rn(fv[j], fx[j], sb[j]);
                    }
                    if (it + i0 + i >= kept_from) {
                        const uint32_t slot = (it + i0 + i - kept_from) * 2 * blockDim.x + tid;
                        kept[slot] = cx[i];
                        kept[slot + blockDim.x] = cv[i];
                    }
                }
#pragma unroll
            for (int i = 0; i < kFlightBwd; ++i) {
                cx[i] = nx[i];
                cv[i] = nv[i];
            }
        }
        float s1[L] = {}, s2[L] = {};
        if (g.cnt) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1[L > 1 ? j : 0] = __fmaf_rn(lanes.w[j], sa[j], s1[L > 1 ? j : 0]);
                s2[L > 1 ? j : 0] = __fmaf_rn(lanes.w[j], sb[j], s2[L > 1 ? j : 0]);
                acc_a[j] += sa[j];
                acc_b[j] += sb[j];
            }
        }
        group_sums<V, L, true>(a, t, s1, s2, g.cnt != 0, s.part, s.warp_sum, s.sum);
        float2* slot = slots + (blockIdx.x + u) * p.gl;
        for (uint32_t q = tid; q < t.groups; q += blockDim.x) slot[q] = s.sum[q];
        it += g.iters;
        w = to;
        if (params && (w == w1 || w / p.rows / a.n != g.tile)) {  // the last segment of the block or of the tile
            channel_sums<V>(t, p.k, acc_a, acc_b, true, s.part, chans + (blockIdx.x + g.tile) * (uint64_t)tile_c);
#pragma unroll
            for (int j = 0; j < V; ++j) acc_a[j] = acc_b[j] = 0.0f;
        }
    }

    cooperative_groups::this_grid().sync();

    const uint32_t lane = tid & 31, warp = tid >> 5;
    const float m = (float)(p.vecs * V / a.groups);
    for (uint64_t end = w1; end > w0;) {
        const uint64_t u = (end - 1) / p.rows, from = u * p.rows > w0 ? u * p.rows : w0;
        Tile t;
        const Segment g = segment_of<V, L>(a, p, u, from, end, t);
        GradLanes<T, V, L> lanes;
        if (g.cnt) {
            lanes.params(a, g.c);
            lanes.stats(a, g.n, g.c);
        }
        __syncthreads();  // s.sum of the segment before is read no more
        for (uint32_t q = warp; q < t.groups; q += blockDim.x / 32) {
            const uint32_t grp = t.g0 + q, t0 = grp * a.per / tile_c, t1 = ((grp + 1) * a.per - 1) / tile_c;
            float s1 = 0.0f, s2 = 0.0f;
            for (uint32_t k = t0; k <= t1; ++k) {
                const uint64_t uu = k * a.n + g.n;
                const uint64_t b0 = uu * p.rows / p.per_block, b1 = ((uu + 1) * p.rows - 1) / p.per_block;
                const uint32_t at = grp - k * tile_c / a.per;
                for (uint64_t b = b0 + lane; b <= b1; b += 32) {
                    const float2 v = __ldcg(slots + (b + uu) * p.gl + at);
                    s1 += v.x;
                    s2 += v.y;
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                s1 += __shfl_xor_sync(~0u, s1, o);
                s2 += __shfl_xor_sync(~0u, s2, o);
            }
            if (lane == 0) s.sum[q] = make_float2(s1, s2);
        }
        __syncthreads();
        it -= g.iters;
        if (g.cnt) {
            GroupGrad<T, V, L> gg;
            gg.take(a, t, g.c, s.sum, m, lanes.rstd);
            const T *x = (const T*)a.x + g.at, *v = (const T*)a.v + g.at;
            T* out = (T*)a.out + g.at;
            for (uint32_t i1 = (g.cnt + kFlightBwd - 1) / kFlightBwd * kFlightBwd; i1 > 0; i1 -= kFlightBwd) {
                Pack<T, V> rx[kFlightBwd], rv[kFlightBwd];
#pragma unroll
                for (int i = kFlightBwd - 1; i >= 0; --i) {
                    const uint32_t k = i1 - kFlightBwd + i;
                    if (k < g.cnt) {
                        if (it + k >= kept_from) {
                            const uint32_t slot = (it + k - kept_from) * 2 * blockDim.x + tid;
                            rx[i] = kept[slot];
                            rv[i] = kept[slot + blockDim.x];
                        } else {
                            rx[i].load(x + (uint64_t)k * step);
                            rv[i].load(v + (uint64_t)k * step);
                        }
                    }
                }
#pragma unroll
                for (int i = kFlightBwd - 1; i >= 0; --i) {
                    const uint32_t k = i1 - kFlightBwd + i;
                    if (k < g.cnt) {
                        float fx[V], fv[V], o[V];
                        rx[i].get(fx);
                        rv[i].get(fv);
                        if (DROP) drop_vector<V>(a.drop, dstep, g.at + (uint64_t)k * step, fv);
                        lanes.template grads<ACT>(fx, fv);
                        gg.apply(lanes, fx, fv, o);
                        rx[i].set(o);
                        rx[i].store(out + (uint64_t)k * step);
                    }
                }
            }
        }
        end = from;
    }
    if (params)
        for (uint32_t ch = blockIdx.x * (blockDim.x / 32) + warp; ch < a.c; ch += gridDim.x * (blockDim.x / 32)) {
            const uint32_t tile = ch / tile_c;
            const uint64_t b0 = tile * a.n * p.rows / p.per_block, b1 = ((tile + 1) * a.n * p.rows - 1) / p.per_block;
            join_channel<T>(a, ch, chans + (b0 + tile) * tile_c + (ch - tile * tile_c), b1 - b0 + 1, tile_c);
        }
}

}  // namespace norm
}  // namespace bsx
