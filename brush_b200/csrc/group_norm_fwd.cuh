// group_norm_fwd.cuh - the forward kernels of group norm.
#pragma once

#include <cooperative_groups.h>

#include "group_norm.cuh"

namespace bsx {
namespace norm {

// What a thread needs of its V channels.
template <class T, int V, int L>
struct Lanes {
    float a[V], b[V], off[L];  // weight rstd, bias, -mean

    __device__ __forceinline__ void load(const Args& g, uint32_t c) {
        params<T, V>(g, g.weight, c, L > 1, 1.0f, a);
        params<T, V>(g, g.bias, c, L > 1, 0.0f, b);
    }
    // stat[q]: mean and rstd of the tile's group q
    __device__ __forceinline__ void fold(const Args& g, const Plan& p, const Tile& t, uint32_t c, const float2* stat) {
        float r[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float2 s = stat[p.by_per(channel_at<L>(g, c, j)) - t.g0];
            off[j] = -s.x;
            r[j] = s.y;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) a[j] *= r[L > 1 ? j : 0];
    }
    template <int ACT>
    __device__ __forceinline__ void apply(float (&v)[V]) const {
        add_v<V>(v, v, off);  // exact for values near the mean: a large mean costs no digits
        fma_v<V>(v, v, a, b);
        activate<ACT>(v);
    }
};

// Small samples: one block per (sample, tile), at most kBatch vectors a thread, held in registers between
// the sums and the result: x is read once. Mean, then the squares of the deviations from it.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) small_fwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    float2* sum = (float2*)smem;           // [gl]
    float2* warp_sum = sum + p.gl;         // [warps]
    float* part = (float*)(((uintptr_t)(warp_sum + kThreads / 32) + 15) & ~(uintptr_t)15);  // places<L>
    float* means = part + places<L>(blockDim.x);  // [gl]
    const uint32_t tid = threadIdx.x;
    const uint32_t n = p.tiles == 1 ? blockIdx.x : blockIdx.x / p.tiles, tile = blockIdx.x - n * p.tiles;
    const Tile t = tile_of<V, L>(a, p, tile);
    const uint32_t row = t.cols == p.cols ? p.by_cols(tid) : tid / t.cols, col = tile * p.cols + tid - row * t.cols;
    const bool active = row < p.k;
    const uint32_t rows = p.rows - (col >= p.last);  // of this column
    const uint32_t step = p.k * p.rv * V;
    const uint64_t at = (n * p.vecs + row * p.rv + col) * V;
    const T* x = (const T*)a.x + at;
    Pack<T, V> raw[kBatch];
    uint32_t cnt = 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (active && row + i * p.k < rows) {
            raw[i].load(x + (uint64_t)i * step);
            cnt = i + 1;
        }
    const uint32_t c = p.tiles > 1 ? col * V : col * V - p.by_c(col * V) * a.c;
    Lanes<T, V, L> lanes;
    if (active) lanes.load(a, c);
    const GroupWalk walk = group_walk<V, L>(a, t, tid);

    constexpr int P = kParts<V, L>;
    const float m = (float)(a.pixels * a.per);  // values of a group
    float acc[P] = {}, val[L], off[L];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
            accumulate<V, P>(acc, f);
        }
    per_item<V, L>(acc, val);
    group_sums<V, L, false>(a, t, walk, val, val, active, part, warp_sum, sum);
#pragma unroll
    for (int j = 0; j < L; ++j) off[j] = active ? -sum[p.by_per(channel_at<L>(a, c, j)) - t.g0].x / m : 0.0f;
    for (uint32_t q = tid; q < t.groups; q += blockDim.x) means[q] = sum[q].x / m;
#pragma unroll
    for (int j = 0; j < P; ++j) acc[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
            add_v<V>(f, f, off);
            accumulate<V, P>(acc, f, f);
        }
    per_item<V, L>(acc, val);
    group_sums<V, L, false>(a, t, walk, val, val, active, part, warp_sum, sum);
    for (uint32_t q = tid; q < t.groups; q += blockDim.x) {
        const float rstd = 1.0f / sqrtf(sum[q].x / m + a.eps);
        sum[q] = make_float2(means[q], rstd);
        a.mean[(uint64_t)n * a.groups + t.g0 + q] = means[q];
        a.rstd[(uint64_t)n * a.groups + t.g0 + q] = rstd;
    }
    __syncthreads();
    if (cnt == 0) return;
    lanes.fold(a, p, t, c, sum);
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

// Large samples: one cooperative launch, each block with a run of rows. Every thread copies its vectors of the
// coming batches of rows into its own places of a ring in shared memory, kAhead batches ahead. First pass: mean and
// sum of squared deviations of each group in each segment (from a pivot, the mean of a thread's first vectors, so
// that no large mean cancels), to the workspace. Grid barrier. Second pass, last row first: the segments' statistics
// are joined, and the rows are normalised out of the ring, which still holds the last ones; the others come again.
template <class T, int V, int L, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads, 1) large_fwd_kernel(const Args a, const Plan p) {
    extern __shared__ float smem[];
    float2* sum = (float2*)smem;                       // [gl]
    float2* warp_sum = sum + p.gl;                     // [warps]
    float2* pivot = warp_sum + kThreads / 32;          // [gl]: mean and count of the block's last segment
    float* part = (float*)(((uintptr_t)(pivot + p.gl) + 15) & ~(uintptr_t)15);  // places<L>, two words a thread at least
    const uint32_t tid = threadIdx.x, threads = blockDim.x;
    Pack<T, V>* ring = (Pack<T, V>*)(((uintptr_t)(part + max(places<L>(threads), 2 * threads)) + 15) & ~(uintptr_t)15) + tid;  // [ring][R][threads]
    constexpr int P = kParts<V, L>, R = kRows, F = kAhead;
    const Run run = run_of(a, p, blockIdx.x);
    const uint64_t step = (uint64_t)run.stride * p.rv * V;
    const uint32_t all = batches_of<R>(p, run);
    float4* slots = (float4*)a.ws;  // [(block + unit) gl + group]: mean, squared deviations, count

    Walk<V, R> ahead;
    ahead.u = run.first;
    ahead.unit(a, p, run, false);
    uint32_t to_slot = 0, slot = 0;  // ring places of the batch to copy and of the batch at work
    const auto copy = [&]() {
        Pack<T, V>* to = ring + to_slot * R * threads;
        const T* x = (const T*)a.x + ahead.at;
        if (ahead.i + R <= ahead.valid) {
#pragma unroll
            for (int j = 0; j < R; ++j) copy_async<T, V>(to + j * threads, x + j * step);
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (ahead.i + j < ahead.valid) copy_async<T, V>(to + j * threads, x + j * step);
        }
    };
#pragma unroll 1
    for (uint32_t b = 0; b < F; ++b) {
        if (b < all) {
            copy();
            ahead.next(a, p, run, step);
            to_slot = to_slot + 1 == p.ring ? 0 : to_slot + 1;
        }
        copy_commit();
    }
    uint32_t batch = 0;
    Tile t;
    Segment g;
    for (uint32_t u = run.first; u <= run.last; ++u) {
        t = tile_of<V, L>(a, p, p.tiles == 1 ? 0 : u / (uint32_t)a.n);
        g = segment_of<V>(a, p, run, u, t);
        const GroupWalk walk = group_walk<V, L>(a, t, tid);
        float off[L] = {}, acc[P] = {}, sq[P] = {};
        const auto take = [&](const Pack<T, V>& v) {
            float f[V];
            v.get(f);
            add_v<V>(f, f, off);
            accumulate<V, P>(acc, f);
            accumulate<V, P>(sq, f, f);
        };
        for (uint32_t i0 = 0; i0 < g.iters; i0 += R, ++batch) {
            copy_wait<F - 1>();
            const Pack<T, V>* at = ring + slot * R * threads;
            if (i0 == 0 && g.cnt) {
                const uint32_t have = min(g.cnt, (uint32_t)R);
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (j < have) {
                        float f[V];
                        at[j * threads].get(f);
                        accumulate<V, P>(acc, f);
                    }
                per_item<V, L>(acc, off);
                const float inv = -1.0f / (float)(have * (V / L));
#pragma unroll
                for (int j = 0; j < L; ++j) off[j] *= inv;
#pragma unroll
                for (int j = 0; j < P; ++j) acc[j] = 0.0f;
            }
            if (i0 + R <= g.cnt) {
#pragma unroll
                for (int j = 0; j < R; ++j) take(at[j * threads]);
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (i0 + j < g.cnt) take(at[j * threads]);
            }
            slot = slot + 1 == p.ring ? 0 : slot + 1;
            if (batch + F < all) {
                copy();
                ahead.next(a, p, run, step);
                to_slot = to_slot + 1 == p.ring ? 0 : to_slot + 1;
            }
            copy_commit();
        }
        const float cnt = (float)g.cnt * (V / L), inv = g.cnt ? 1.0f / cnt : 0.0f;
        float mean[L], dev[L], val[L], s[L], s2[L];
        per_item<V, L>(acc, s);
        per_item<V, L>(sq, s2);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float d = s[j] * inv;
            mean[j] = d - off[j];
            dev[j] = __fmaf_rn(-s[j], d, s2[j]);
            if (dev[j] < 0.0f) dev[j] = 0.0f;  // rounding; NaN stays
            val[j] = cnt * mean[j];
        }
        group_sums<V, L, false>(a, t, walk, val, val, g.cnt != 0, part, warp_sum, sum);
        for (uint32_t q = tid; q < t.groups; q += threads) {
            uint32_t lo, hi;
            group_span<V, V>(a, t, q, lo, hi);
            const float count = g.pixels * (float)(hi - lo);
            pivot[q] = make_float2(sum[q].x / count, count);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < L; ++j) {
            val[j] = 0.0f;
            if (g.cnt) {
                const float d = mean[j] - pivot[p.by_per(channel_at<L>(a, g.c, j)) - t.g0].x;
                val[j] = __fmaf_rn(cnt * d, d, dev[j]);
            }
        }
        group_sums<V, L, false>(a, t, walk, val, val, g.cnt != 0, part, warp_sum, sum);
        for (uint32_t q = tid; q < t.groups; q += threads)
            slots[(uint64_t)(blockIdx.x + u) * p.gl + q] = make_float4(pivot[q].x, sum[q].x, pivot[q].y, 0.0f);
    }

    // What the second pass needs and no other block gives.
    const uint32_t dstep = DROP ? drop_step(a.drop) : 0u;
    const float m = (float)(a.pixels * a.per);
    const uint32_t resident = all > p.ring ? all - p.ring : 0;  // batches from here on are in the ring
    uint32_t next = all - 1;                                    // the batch that `ahead` is at
    ahead.u = run.last;
    ahead.unit(a, p, run, true);
    while (next >= resident && next > 0) {
        ahead.before(a, p, run, step);
        --next;
    }
    slot = (all - 1) % p.ring;
    to_slot = next % p.ring;
    Lanes<T, V, L> lanes;
    if (g.cnt) lanes.load(a, g.c);

    cooperative_groups::this_grid().sync();

    for (uint32_t u = run.last;; --u) {
        if (u != run.last) {
            t = tile_of<V, L>(a, p, p.tiles == 1 ? 0 : u / (uint32_t)a.n);
            g = segment_of<V>(a, p, run, u, t);
            if (g.cnt) lanes.load(a, g.c);
            __syncthreads();  // sum and pivot are read no more
            for (uint32_t q = tid; q < t.groups; q += threads)
                pivot[q].x = __ldcg(slots + (uint64_t)(blockIdx.x + u) * p.gl + q).x;
            __syncthreads();
        }
        // Joined about a pivot, the mean of this block's own segment: its share of the values bounds how far off it is.
        join_runs<V>(a, p, t, g.n, part, sum, [&](uint64_t i, uint32_t q, float& s, float& s2) {
            const float4 v = __ldcg(slots + i);
            const float d = v.x - pivot[q].x;
            s = __fmaf_rn(v.z, d, s);
            s2 += __fmaf_rn(v.z * d, d, v.y);
        });
        for (uint32_t q = tid; q < t.groups; q += threads) {
            const uint32_t grp = t.g0 + q;
            const float d = sum[q].x / m, mean = pivot[q].x + d;
            float dev = __fmaf_rn(-sum[q].x, d, sum[q].y);
            if (dev < 0.0f) dev = 0.0f;
            const float rstd = 1.0f / sqrtf(dev / m + a.eps);
            sum[q] = make_float2(mean, rstd);
            if (g.r0 == 0 && grp * a.per >= t.c0) {
                a.mean[(uint64_t)g.n * a.groups + grp] = mean;
                a.rstd[(uint64_t)g.n * a.groups + grp] = rstd;
            }
        }
        __syncthreads();
        if (g.cnt) lanes.fold(a, p, t, g.c, sum);
        uint64_t at = g.at + (g.iters - 1) / R * R * step;
        const auto give = [&](const Pack<T, V>& v, uint64_t where) {
            float f[V];
            v.get(f);
            lanes.template apply<ACT>(f);
            if (DROP) drop_vector<V>(a.drop, dstep, where, f);
            Pack<T, V> o;
            o.set(f);
            o.store((T*)a.out + where);
        };
        for (uint32_t i0 = (g.iters - 1) / R * R;; i0 -= R) {
            --batch;
            copy_wait<F - 1>();
            const Pack<T, V>* have = ring + slot * R * threads;
            if (i0 + R <= g.cnt) {
#pragma unroll
                for (int j = 0; j < R; ++j) give(have[j * threads], at + j * step);
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (i0 + j < g.cnt) give(have[j * threads], at + j * step);
            }
            at -= R * step;
            slot = slot == 0 ? p.ring - 1 : slot - 1;
            if (batch == next + F && next < resident) {
                copy();
                to_slot = to_slot == 0 ? p.ring - 1 : to_slot - 1;
                if (next > 0) {
                    ahead.before(a, p, run, step);
                    --next;
                }
            }
            copy_commit();
            if (i0 == 0) break;
        }
        if (u == run.first) break;
    }
}

}  // namespace norm
}  // namespace bsx
