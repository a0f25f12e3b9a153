// group_norm_fwd.cuh - the forward kernels of group norm.
#pragma once

#include <cooperative_groups.h>

#include <utility>

#include "group_norm.cuh"

namespace bsx {
namespace norm {

// What a thread needs of its V channels.
template <class T, int V, int L>
struct Lanes {
    float a[V], b[V], off[L];  // weight rstd, bias, -mean

    __device__ __forceinline__ void load(const Args& g, uint32_t c) {
        params<T, V>(g, g.weight, c, 1.0f, a);
        params<T, V>(g, g.bias, c, 0.0f, b);
    }
    // stat[q]: mean and rstd of the tile's group q
    __device__ __forceinline__ void fold(const Args& g, const Plan& p, const Tile& t, uint32_t c, const float2* stat) {
        float r[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float2 s = stat[p.by_per(channel_at<V, L>(g, c, j)) - t.g0];
            off[j] = -s.x;
            r[j] = s.y;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) a[j] *= r[j * L / V];
    }
    __device__ __forceinline__ void apply(int act, float (&v)[V]) const {
        add_v<V>(v, v, off);  // exact for values near the mean: a large mean costs no digits
        fma_v<V>(v, v, a, b);
        activate<V>(act, v);
    }
};

// Small samples: one block per (sample, tile), at most kBatch vectors a thread, held in registers between
// the sums and the result: x is read once. Mean, then the squares of the deviations from it. Latency bounds it (the
// loads, two sums of three barriers each): one 16 x 16 x 32 float sample 5.6 us, 2048 vectors of 512 f16 channels
// 6.2 us. Two blocks of 512 threads an SM (64 registers, a few spills) against one: 6.0 and 8.1 us for the latter.
template <class T, int V, int L, int ACT, int DROP>
__global__ void __launch_bounds__(kThreads, 2) small_fwd_kernel(const Plan p, const Args a) {
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
    const uint64_t at = n * p.elems + (uint64_t)(row * p.rv + col) * V;
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
            accumulate<V, L>(acc, f);
        }
    per_item<V, L>(acc, val);
    group_sums<V, L, false>(a, t, walk, val, val, active, part, warp_sum, sum);
#pragma unroll
    for (int j = 0; j < L; ++j) off[j] = active ? -sum[p.by_per(channel_at<V, L>(a, c, j)) - t.g0].x / m : 0.0f;
    for (uint32_t q = tid; q < t.groups; q += blockDim.x) means[q] = sum[q].x / m;
#pragma unroll
    for (int j = 0; j < P; ++j) acc[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
            add_v<V>(f, f, off);
            accumulate<V, L>(acc, f, f);
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
    const uint32_t dstep = drops<DROP>(a) ? drop_step(a.drop) : 0u;
    T* out = (T*)a.out + at;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < cnt) {
            float f[V];
            raw[i].get(f);
            lanes.apply(act_of<ACT>(a), f);
            if (drops<DROP>(a)) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, f);
            raw[i].set(f);
            raw[i].store(out + (uint64_t)i * step);
        }
}

// Large samples: one cooperative launch. Every thread copies its vectors of the block's coming batches of rows into
// its own places of a ring in shared memory, some batches ahead. First pass: mean and sum of squared deviations of
// each group in each segment, to the workspace. Deviations are taken from a pivot, the group's mean over the block's
// first batch, so that no large mean cancels (what the pivot is off by enters the sum of squares at most a batch's
// share of the block's rows times over). Grid barrier. Second pass, last row first: the segments' statistics are joined, and the rows are
// normalised out of the ring, which still holds the last ones; the others come again.
// A full frame of 64 bf16 channels (265 MB, larger than L2) takes 136 us: 27 MB stay in the rings, so 482 MB are read
// from DRAM (measured; some 20 MB hit L2) and 265 MB written (213 of them before the kernel ends, the others are in L2
// then): 5.5 TB/s, 84 % of the measured copy rate; read once and written once it would be 81 us. Keeping more in L2
// (evict_last, prefetches between the passes) gave 3 % at most; deeper rings, bulk copies and other batch sizes
// nothing. 8 x 64 x 64 x 256 (17 MB, all of it stays) takes 15.5 us against 5.1: 5 us until the last row has arrived,
// 1 for the sums, 1.5 each for the barrier and the join, 4 for the second pass, which the special-function unit
// bounds (three uses for two elements, four lanes a cycle and scheduler), the rest launch and prologue.
template <class T, int V, int L, int ACT, int DROP, bool S>
__global__ void __launch_bounds__(kThreads, 1) large_fwd_kernel(const Plan p, const Args a) {
    extern __shared__ float smem[];
    float2* sum = (float2*)smem;                       // [gl]
    float2* warp_sum = sum + p.gl;                     // [warps]
    float* pivot = (float*)(warp_sum + kThreads / 32);  // [gl]: later the mean of the block's segment
    float* part = (float*)(((uintptr_t)(pivot + p.gl) + 15) & ~(uintptr_t)15);  // [2] places<L>
    const uint32_t tid = threadIdx.x, threads = blockDim.x;
    Pack<T, V>* ring = (Pack<T, V>*)(((uintptr_t)(part + 2 * places<L>(threads)) + 15) & ~(uintptr_t)15) + tid;  // [ring][R][E][threads]
    constexpr int P = kParts<V, L>, R = rows_of_batch(false, S), F = batches_ahead(false, S), E = S ? 2 : 1;
    const Run run = run_of(a, p);
    const uint64_t step = (uint64_t)run.stride * p.rv * V;
    const uint32_t all = batches_of<R>(p, run);
    const uint64_t count = a.n * p.elems;
    float2* slots = (float2*)a.ws;  // [(block + unit) gl + group]: mean, squared deviations

    Walk<V, R> ahead;
    ahead.u = run.first;
    ahead.unit(a, p, run, false);
    uint32_t to_slot = 0, slot = 0;  // ring places of the batch to copy and of the batch at work
    const auto copy = [&]() {
        Pack<T, V>* to = ring + to_slot * R * E * threads;
        if (ahead.i + R <= ahead.valid) {
#pragma unroll
            for (int j = 0; j < R; ++j) copy_vector<T, V, S>(to + j * E * threads, (const T*)a.x, ahead.at + j * step, count);
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (ahead.i + j < ahead.valid) copy_vector<T, V, S>(to + j * E * threads, (const T*)a.x, ahead.at + j * step, count);
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
        float off[L], acc[P] = {}, sq[P] = {}, all_acc[P] = {}, all_sq[P] = {}, val[L], val2[L];
        copy_wait<F - 1>();
        {
            const Pack<T, V>* at = ring + slot * R * E * threads;
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (j < g.cnt) {
                    float f[V];
                    read_vector<T, V, S>(at + j * E * threads, g.at + j * step).get(f);
                    if (S && j + 1 == g.tail) cut<V>(f, p.tail);
                    accumulate<V, L>(acc, f);
                }
            per_item<V, L>(acc, val);
            group_sums<V, L, false>(a, t, walk, val, val, g.cnt != 0, part, warp_sum, sum);
            const Rows few = {0, min(g.iters, (uint32_t)R), g.rows.ends && g.iters <= R};
            const float pixels = pixels_of(p, few);
            for (uint32_t q = tid; q < t.groups; q += threads) {
                uint32_t lo, hi;
                group_span<V, V>(a, t, q, lo, hi);
                // in the values' own type: differences from it have few digits, and a long sum of them rounds rarely,
                // instead of by the same amount at each addition
                pivot[q] = to_f(from_f<T>(sum[q].x / (pixels * (float)(hi - lo))));
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < L; ++j) off[j] = g.cnt ? -pivot[p.by_per(channel_at<V, L>(a, g.c, j)) - t.g0] : 0.0f;
#pragma unroll
            for (int j = 0; j < P; ++j) acc[j] = 0.0f;
        }
        const auto take = [&](const Pack<T, V>& v, uint32_t i) {
            float f[V];
            v.get(f);
            add_v<V>(f, f, off);
            if (S && i + 1 == g.tail) cut<V>(f, p.tail);
            accumulate<V, L>(acc, f);
            accumulate<V, L>(sq, f, f);
        };
        for (uint32_t i0 = 0; i0 < g.iters; i0 += R, ++batch) {
            copy_wait<F - 1>();
            const Pack<T, V>* at = ring + slot * R * E * threads;
            if (i0 + R <= g.cnt) {
#pragma unroll
                for (int j = 0; j < R; ++j) take(read_vector<T, V, S>(at + j * E * threads, g.at + (i0 + j) * step), i0 + j);
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (i0 + j < g.cnt) take(read_vector<T, V, S>(at + j * E * threads, g.at + (i0 + j) * step), i0 + j);
            }
            slot = slot + 1 == p.ring ? 0 : slot + 1;
            if (batch + F < all) {
                copy();
                ahead.next(a, p, run, step);
                to_slot = to_slot + 1 == p.ring ? 0 : to_slot + 1;
            }
            copy_commit();
            if (i0 / R % 16 == 15 || i0 + R >= g.iters) {  // sums of sums: no chain grows with the sample
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    all_acc[j] += acc[j];
                    all_sq[j] += sq[j];
                    acc[j] = sq[j] = 0.0f;
                }
            }
        }
        per_item<V, L>(all_acc, val);
        per_item<V, L>(all_sq, val2);
        group_sums<V, L, true>(a, t, walk, val, val2, g.cnt != 0, part, warp_sum, sum);
        const float pixels = pixels_of(p, g.rows);
        for (uint32_t q = tid; q < t.groups; q += threads) {
            uint32_t lo, hi;
            group_span<V, V>(a, t, q, lo, hi);
            const float2 s = sum[q];
            const float d = s.x / (pixels * (float)(hi - lo));
            float dev = __fmaf_rn(-s.x, d, s.y);
            if (dev < 0.0f) dev = 0.0f;  // rounding; NaN stays
            pivot[q] += d;
            slots[(uint64_t)(block_id() + u) * p.gl + q] = make_float2(pivot[q], dev);
        }
    }

    const cooperative_groups::grid_group grid = cooperative_groups::this_grid();
    auto arrived = grid.barrier_arrive();
    // What the second pass needs and no other block gives.
    const uint32_t dstep = drops<DROP>(a) ? drop_step(a.drop) : 0u;
    const float m = (float)(a.pixels * a.per);
    const uint32_t resident = all > p.ring ? all - p.ring : 0;  // batches from here on are in the ring
    uint32_t next = resident ? resident - 1 : 0;                // the batch that `ahead` is at
    ahead.rewind(a, p, run, step, all, next);
    slot = (all - 1) % p.ring;
    to_slot = next % p.ring;
    Lanes<T, V, L> lanes;
    if (g.cnt) lanes.load(a, g.c);
    grid.barrier_wait(std::move(arrived));

    for (uint32_t u = run.last;; --u) {
        if (u != run.last) {
            t = tile_of<V, L>(a, p, p.tiles == 1 ? 0 : u / (uint32_t)a.n);
            g = segment_of<V>(a, p, run, u, t);
            if (g.cnt) lanes.load(a, g.c);
            __syncthreads();  // sum and pivot are read no more
            for (uint32_t q = tid; q < t.groups; q += threads) pivot[q] = __ldcg(slots + (uint64_t)(block_id() + u) * p.gl + q).x;
            __syncthreads();
        }
        // Joined about a pivot, the mean of this block's own segment: its share of the values bounds how far off it is.
        join_runs<V>(a, p, t, g.n, slots, part, sum, [&](float2 v, float count, uint32_t q, float& s, float& s2) {
            const float d = v.x - pivot[q];
            s = __fmaf_rn(count, d, s);
            s2 += __fmaf_rn(count * d, d, v.y);
        });
        for (uint32_t q = tid; q < t.groups; q += threads) {
            const uint32_t grp = t.g0 + q;
            const float d = sum[q].x / m, mean = pivot[q] + d;
            float dev = __fmaf_rn(-sum[q].x, d, sum[q].y);
            if (dev < 0.0f) dev = 0.0f;
            const float rstd = 1.0f / sqrtf(dev / m + a.eps);
            sum[q] = make_float2(mean, rstd);
            if (g.rows.r0 == 0 && grp * a.per >= t.c0) {
                a.mean[(uint64_t)g.n * a.groups + grp] = mean;
                a.rstd[(uint64_t)g.n * a.groups + grp] = rstd;
            }
        }
        __syncthreads();
        if (g.cnt) lanes.fold(a, p, t, g.c, sum);
        uint64_t at = g.at + (g.iters - 1) / R * R * step;
        const auto give = [&](const Pack<T, V>& v, uint64_t where, bool cut_short) {
            float f[V];
            v.get(f);
            if (S && cut_short) cut<V>(f, p.tail);  // two lanes share a reciprocal, and so its rounding
            lanes.apply(act_of<ACT>(a), f);
            if (drops<DROP>(a)) drop_vector<V, S>(a.drop, dstep, where, f);
            Pack<T, V> o;
            o.set(f);
            return o;
        };
        for (uint32_t i0 = (g.iters - 1) / R * R;; i0 -= R) {
            --batch;
            copy_wait<F - 1>();
            const Pack<T, V>* have = ring + slot * R * E * threads;
            if constexpr (S) {
#pragma unroll
                for (int j = 0; j < R; ++j) {  // all threads: neighbours exchange what they store
                    const uint64_t where = at + j * step;
                    const bool ok = i0 + j < g.cnt;
                    Pack<T, V> o{};
                    const bool cut_short = i0 + j + 1 == g.tail;
                    if (ok) o = give(read_vector<T, V, S>(have + j * E * threads, where), where, cut_short);
                    store_shifted<T, V>((T*)a.out, where, o, ok, cut_short ? p.tail : V);
                }
            } else if (i0 + R <= g.cnt) {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    give(read_vector<T, V, S>(have + j * threads, at + j * step), at + j * step, false).store((T*)a.out + at + j * step);
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (i0 + j < g.cnt)
                        give(read_vector<T, V, S>(have + j * threads, at + j * step), at + j * step, false).store((T*)a.out + at + j * step);
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
