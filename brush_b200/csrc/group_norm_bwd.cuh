// group_norm_bwd.cuh - the backward kernels of group norm.
#pragma once

#include "group_norm_fwd.cuh"

namespace bsx {
namespace norm {

// With d = x - mean: z = (gamma rstd) d + beta, xh = rstd d, and
//   v_x = rstd (gamma dz - s1 - xh s2) = (gamma rstd) dz - u1 - rstd^2 u2 d,
// u1 and u2 being the group's sums of (gamma rstd) dz and (gamma rstd) dz d over its number of values.
// What a thread needs of its V channels:
template <class T, int V, int L>
struct GradLanes {
    float w[V], b[V], off[L], rstd[L];  // gamma rstd, beta, -mean

    __device__ __forceinline__ void load(const Args& a, uint32_t c) {
        params<T, V>(a, a.weight, c, 1.0f, w);
        params<T, V>(a, a.bias, c, 0.0f, b);
        if (a.act == BSX_ACT_GELU_TANH) {
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = near_bias(b[j]);
        }
    }
    __device__ __forceinline__ void stats(const Args& a, const Plan& p, uint64_t n, uint32_t c) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const uint64_t at = n * a.groups + p.by_per(channel_at<V, L>(a, c, j));
            off[j] = -__ldg(a.mean + at);
            rstd[j] = __ldg(a.rstd + at);
        }
    }
    __device__ __forceinline__ void scale(float (&to)[V], const float (&gamma)[V]) const { mul_v<V>(to, gamma, rstd); }
    // x becomes d, v becomes dz
    __device__ __forceinline__ void grads(int act, float (&x)[V], float (&v)[V]) const {
        add_v<V>(x, x, off);
        float z[V];
        fma_v<V>(z, x, w, b);
        back_activate<V>(act, v, z);
    }
};

template <class T, int V, int L>
struct GroupGrad {
    float u1[L], u2[L];  // -u1, -rstd^2 u2
    __device__ __forceinline__ void take(const Args& g, const Plan& p, const Tile& t, uint32_t c, const float2* sum, float m,
                                         const GradLanes<T, V, L>& lanes) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const float2 s = sum[p.by_per(channel_at<V, L>(g, c, j)) - t.g0];
            u1[j] = -s.x / m;
            u2[j] = -s.y / m * lanes.rstd[j] * lanes.rstd[j];
        }
    }
    // d becomes v_x
    __device__ __forceinline__ void apply(const GradLanes<T, V, L>& lanes, float (&d)[V], const float (&dz)[V]) const {
        fma_v<V>(d, d, u2, u1);
        fma_v<V>(d, lanes.w, dz, d);
    }
};

// Rows (of large samples) or samples (small ones) after which a thread's sums go into sums of sums, so that no chain
// of additions grows with the tensor: a gradient that is the same everywhere would round the same way each time.
// 33.5 M pixels of 64 floats, 0.9 each: v_bias off by 1100 half steps without.
constexpr uint32_t kSumRows = 64;

// Into a thread's own places: x, or x more; x starts again.
template <int V>
__device__ __forceinline__ void lay_by(float* part, float (&x)[V], bool more) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float& at = part[place<V>(threadIdx.x * V + j)];
        at = more ? at + x[j] : x[j];
        x[j] = 0.0f;
    }
}
template <int V>
__device__ __forceinline__ void take_back(const float* part, float (&x)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] += part[place<V>(threadIdx.x * V + j)];
}

// A block's sums over its copies of each channel of a tile (x and y: one value an element), in a fixed order,
// to to[channel - c0], or added there. Starts without a barrier like group_sums, ends with one.
template <int V>
__device__ __forceinline__ void channel_sums(const Tile& t, uint32_t items, const float (&x)[V], const float (&y)[V],
                                             bool active, float* part, float2* to, bool more = false) {
    const uint32_t tid = threadIdx.x, half = places<V>(blockDim.x);
    const uint32_t width = t.c1 - t.c0, copies = items * V / width;
    put_items<V>(part, x, active);
    put_items<V>(part + half, y, active);
    __syncthreads();
    // q threads a channel sum every q-th copy into the first q copies, then one adds those
    uint32_t q = min(blockDim.x / width, copies);
    if (q > 1) {
        const uint32_t z = tid / width, i = tid - z * width;
        if (z < q) {
            float s = 0.0f, s2 = 0.0f;
#pragma unroll 4
            for (uint32_t m = z; m < copies; m += q) {
                const uint32_t at = place<V>(m * width + i);
                s += part[at];
                s2 += part[half + at];
            }
            const uint32_t at = place<V>(z * width + i);
            part[at] = s;
            part[half + at] = s2;
        }
        __syncthreads();
    } else {
        q = copies;
    }
    for (uint32_t i = tid; i < width; i += blockDim.x) {
        float s = 0.0f, s2 = 0.0f;
#pragma unroll 4
        for (uint32_t m = 0; m < q; ++m) {
            const uint32_t at = place<V>(m * width + i);
            s += part[at];
            s2 += part[half + at];
        }
        if (more) s += to[i].x, s2 += to[i].y;
        to[i] = make_float2(s, s2);
    }
    __syncthreads();
}

// Parameter gradients of one channel from its partial sums (x: bias, y: weight), by a warp.
template <class T>
__device__ __forceinline__ void join_channel(const Args& a, uint32_t c, const float2* from, uint32_t count,
                                             uint64_t stride) {
    float s = 0.0f, s2 = 0.0f;
    constexpr int G = 4;  // loads in flight
    for (uint32_t i = threadIdx.x & 31; i < count; i += G * 32) {
        float2 v[G];
#pragma unroll
        for (int k = 0; k < G; ++k) v[k] = i + k * 32 < count ? __ldcg(from + (i + k * 32) * stride) : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < G; ++k) {
            s += v[k].x;
            s2 += v[k].y;
        }
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
template <class T, int V, int L, int ACT, int DROP>
__global__ void __launch_bounds__(kThreads) small_bwd_kernel(const Plan p, const Args a) {
    extern __shared__ float smem[];
    float2* sum = (float2*)smem;                       // [gl]
    float2* warp_sum = sum + p.gl;                     // [warps]
    float* part = (float*)(((uintptr_t)(warp_sum + kThreads / 32) + 15) & ~(uintptr_t)15);  // [2] places<V>
    constexpr int P = kParts<V, L>;
    const uint32_t tid = threadIdx.x, tile = blockIdx.x % p.tiles;
    const Tile t = tile_of<V, L>(a, p, tile);
    const uint32_t row = t.cols == p.cols ? p.by_cols(tid) : tid / t.cols, col = tile * p.cols + tid - row * t.cols;
    const bool active = row < p.k;
    const uint32_t rows = p.rows - (col >= p.last);
    const uint32_t step = p.k * p.rv * V;
    uint32_t cnt = 0;
#pragma unroll
    for (int i = 0; i < kBatchBwd; ++i)
        if (active && row + i * p.k < rows) cnt = i + 1;
    const uint32_t c = p.tiles > 1 ? col * V : col * V - p.by_c(col * V) * a.c;
    const uint32_t dstep = drops<DROP>(a) ? drop_step(a.drop) : 0u;
    const float m = (float)(a.pixels * a.per);
    GradLanes<T, V, L> lanes;
    float gamma[V];
    if (active) lanes.load(a, c);
#pragma unroll
    for (int j = 0; j < V; ++j) gamma[j] = lanes.w[j];
    const GroupWalk walk = group_walk<V, L>(a, t, tid);
    float acc_a[V] = {}, acc_b[V] = {};
    float2* const mine = (float2*)a.ws + (uint64_t)(blockIdx.x / p.tiles) * a.c + t.c0;
    const bool wanted = a.v_weight || a.v_bias;  // of all blocks alike
    uint32_t done = 0;                           // samples
    for (uint32_t n = blockIdx.x / p.tiles; n < a.n; n += gridDim.x / p.tiles) {
        const uint64_t at = n * p.elems + (uint64_t)(row * p.rv + col) * V;
        Pack<T, V> rx[kBatchBwd], rv[kBatchBwd];
#pragma unroll
        for (int i = 0; i < kBatchBwd; ++i)
            if (i < cnt) {
                rx[i].load((const T*)a.x + at + (uint64_t)i * step);
                rv[i].load((const T*)a.v + at + (uint64_t)i * step);
            }
        if (active) {
            lanes.stats(a, p, n, c);
            lanes.scale(lanes.w, gamma);
        }
        float s1[P] = {}, s2[P] = {};
#pragma unroll
        for (int i = 0; i < kBatchBwd; ++i)
            if (i < cnt) {
                float x[V], v[V];
                rx[i].get(x);
                rv[i].get(v);
                if (drops<DROP>(a)) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, v);
                lanes.grads(act_of<ACT>(a), x, v);
                accumulate<V, V>(acc_a, v);
                float t1[V];
                mul_v<V>(t1, x, lanes.rstd);
                accumulate<V, V>(acc_b, v, t1);
                mul_v<V>(v, v, lanes.w);
                accumulate<V, L>(s1, v);
                accumulate<V, L>(s2, v, x);
            }
        float i1[L], i2[L];
        per_item<V, L>(s1, i1);
        per_item<V, L>(s2, i2);
        group_sums<V, L, true>(a, t, walk, i1, i2, active, part, warp_sum, sum);
        if (cnt) {
            GroupGrad<T, V, L> gg;
            gg.take(a, p, t, c, sum, m, lanes);
#pragma unroll
            for (int i = 0; i < kBatchBwd; ++i)
                if (i < cnt) {
                    float x[V], v[V];
                    rx[i].get(x);
                    rv[i].get(v);
                    if (drops<DROP>(a)) drop_vector<V>(a.drop, dstep, at + (uint64_t)i * step, v);
                    lanes.grads(act_of<ACT>(a), x, v);
                    gg.apply(lanes, x, v);
                    rx[i].set(x);
                    rx[i].store((T*)a.out + at + (uint64_t)i * step);
                }
        }
        // sum is read above and written again only after the next call's first barrier
        if (++done % kSumRows == 0 && wanted) {
            channel_sums<V>(t, p.k * t.cols, acc_a, acc_b, active, part, mine, done > kSumRows);
#pragma unroll
            for (int j = 0; j < V; ++j) acc_a[j] = acc_b[j] = 0.0f;
        }
    }
    if (!wanted) return;
    const float2* ws = (const float2*)a.ws;
    __syncthreads();
    channel_sums<V>(t, p.k * t.cols, acc_a, acc_b, active, part, mine, done >= kSumRows);
    cooperative_groups::this_grid().sync();
    for (uint32_t ch = blockIdx.x * (blockDim.x / 32) + tid / 32; ch < a.c; ch += gridDim.x * (blockDim.x / 32))
        join_channel<T>(a, ch, ws + ch, gridDim.x / p.tiles, a.c);
}

// Large samples: runs and rings like the forward's, a ring for x and one for v. First pass: a thread's sums of dz and
// dz d of each of its channels in a segment, from which come the segment's sums of each group and the block's of each
// channel, to the workspace. Grid barrier. Second pass, last row first: the group sums are joined and v_x formed; then
// the channels are dealt to the warps of the grid.
// A half-resolution frame of 128 bf16 channels (133 MB each of x, v and v_x) takes 110 us: 27 MB stay in the rings,
// 468 MB are read from DRAM (measured; some 36 MB hit L2) and 133 MB written (83 before the kernel ends), 5.5 TB/s, 84 %
// of the measured copy rate; read and written once it would be 61 us. 8 x 64 x 64 x 256 takes 23 us against 7.7: 9 us
// for the first pass (34 MB, with two special-function uses and about 90 FP32 operations a vector lane), 5 for sums,
// barrier and join, 6 for the second pass, 1 to 2 for the channels.
template <class T, int V, int L, int ACT, int DROP, bool S>
__global__ void __launch_bounds__(kThreads, 1) large_bwd_kernel(const Plan p, const Args a) {
    extern __shared__ float smem[];
    constexpr int P = kParts<V, L>, R = rows_of_batch(true, S), F = batches_ahead(true, S), E = S ? 2 : 1;
    const uint32_t tid = threadIdx.x, threads = blockDim.x, tile_c = p.tiles == 1 ? a.c : p.cols * V;
    float2* sum = (float2*)smem;            // [gl]
    float2* warp_sum = sum + p.gl;          // [warps]
    float2* chan = warp_sum + kThreads / 32;  // [tile_c]
    float* part = (float*)(((uintptr_t)(chan + tile_c) + 15) & ~(uintptr_t)15);  // [2] places<V>
    Pack<T, V>* ring = (Pack<T, V>*)(((uintptr_t)(part + 2 * places<V>(threads)) + 15) & ~(uintptr_t)15) + tid;  // [ring][R][x, v][E][threads]
    const Run run = run_of(a, p);
    const uint64_t step = (uint64_t)run.stride * p.rv * V;
    const uint32_t all = batches_of<R>(p, run);
    const uint32_t resident = all > p.ring ? all - p.ring : 0;  // batches from here on are in the ring after the first pass
    const uint32_t dstep = drops<DROP>(a) ? drop_step(a.drop) : 0u;
    const float scale[1] = {a.drop.scale};
    float2* slots = (float2*)a.ws;                                                   // [(block + unit) gl + group]
    float2* chans = slots + (uint64_t)(gridDim.x * gridDim.y + p.tiles * (uint32_t)a.n) * p.gl;  // [(block + tile) tile_c + channel - c0]
    const bool wanted = a.v_weight || a.v_bias;
    const uint64_t count = a.n * p.elems;

    Walk<V, R> ahead;
    ahead.u = run.first;
    ahead.unit(a, p, run, false);
    uint32_t to_slot = 0, slot = 0;
    const auto copy = [&]() {
        Pack<T, V>* to = ring + to_slot * 2 * R * E * threads;
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (ahead.i + j < ahead.valid) {
                copy_vector<T, V, S>(to + 2 * j * E * threads, (const T*)a.x, ahead.at + j * step, count);
                copy_vector<T, V, S>(to + (2 * j + 1) * E * threads, (const T*)a.v, ahead.at + j * step, count);
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
    Segment g{};
    GradLanes<T, V, L> lanes;
    uint32_t kept_tile = ~0u;  // the tile that the block has sums of channels for: a segment's are added to them
    float sa[V], sb[V];
    for (uint32_t u = run.first; u <= run.last; ++u) {
        t = tile_of<V, L>(a, p, p.tiles == 1 ? 0 : u / (uint32_t)a.n);
        g = segment_of<V>(a, p, run, u, t);
        if (g.cnt) {
            lanes.load(a, g.c);
            lanes.stats(a, p, g.n, g.c);
            lanes.scale(lanes.w, lanes.w);
        }
        const GroupWalk walk = group_walk<V, L>(a, t, tid);
#pragma unroll
        for (int j = 0; j < V; ++j) sa[j] = sb[j] = 0.0f;
        uint64_t at = g.at;
        const auto take = [&](const Pack<T, V>* px, Pack<T, V>* in, uint64_t where, bool cut_short) {
            float fx[V], fv[V];
            Pack<T, V> pv = read_vector<T, V, S>(in, where);
            read_vector<T, V, S>(px, where).get(fx);
            if (drops<DROP>(a)) {
                drop_packed<S>(a.drop, dstep, where, pv);
                if (!S && batch >= resident) {  // the second pass need not draw again
                    if (V * sizeof(T) == 2) pv.w[0] |= pv.w[0] << 16;
                    *in = pv;
                }
            }
            pv.get(fv);
            if (S && cut_short) {  // two lanes share a reciprocal, and so its rounding
                cut<V>(fx, p.tail);
                cut<V>(fv, p.tail);
            }
            if (drops<DROP>(a)) mul_v<V>(fv, fv, scale);
            lanes.grads(act_of<ACT>(a), fx, fv);
            if (S && cut_short) {
                cut<V>(fx, p.tail);
                cut<V>(fv, p.tail);
            }
            accumulate<V, V>(sa, fv);
            accumulate<V, V>(sb, fv, fx);
        };
        for (uint32_t from = 0; from < g.iters; from += kSumRows) {
            const uint32_t stop = min(g.iters, from + kSumRows);
            for (uint32_t i0 = from; i0 < stop; i0 += R, ++batch) {
                copy_wait<F - 1>();
                Pack<T, V>* have = ring + slot * 2 * R * E * threads;
                if (i0 + R <= g.cnt) {
#pragma unroll
                    for (int j = 0; j < R; ++j) take(have + 2 * j * E * threads, have + (2 * j + 1) * E * threads, at + j * step, i0 + j + 1 == g.tail);
                } else {
#pragma unroll
                    for (int j = 0; j < R; ++j)
                        if (i0 + j < g.cnt) take(have + 2 * j * E * threads, have + (2 * j + 1) * E * threads, at + j * step, i0 + j + 1 == g.tail);
                }
                at += R * step;
                slot = slot + 1 == p.ring ? 0 : slot + 1;
                if (batch + F < all) {
                    copy();
                    ahead.next(a, p, run, step);
                    to_slot = to_slot + 1 == p.ring ? 0 : to_slot + 1;
                }
                copy_commit();
            }
            if (stop < g.iters) {  // part is free until group_sums
                lay_by<V>(part, sa, from > 0);
                lay_by<V>(part + places<V>(threads), sb, from > 0);
            }
        }
        if (g.iters > kSumRows) {
            take_back<V>(part, sa);
            take_back<V>(part + places<V>(threads), sb);
            __syncthreads();  // group_sums writes over others' places
        }
        float s1[P] = {}, s2[P] = {}, i1[L], i2[L];
        if (g.cnt) {
            accumulate<V, L>(s1, sa, lanes.w);
            accumulate<V, L>(s2, sb, lanes.w);
        }
        per_item<V, L>(s1, i1);
        per_item<V, L>(s2, i2);
        group_sums<V, L, true>(a, t, walk, i1, i2, g.cnt != 0, part, warp_sum, sum);
        for (uint32_t q = tid; q < t.groups; q += threads) slots[(uint64_t)(block_id() + u) * p.gl + q] = sum[q];
        if (wanted) {
            mul_v<V>(sb, sb, lanes.rstd);
            channel_sums<V>(t, t.cols, sa, sb, g.cnt != 0, part, chan);
            float2* to = chans + (uint64_t)(block_id() + g.tile) * tile_c;
            for (uint32_t i = tid; i < t.c1 - t.c0; i += threads) {
                float2 s = chan[i];
                if (kept_tile == g.tile) {
                    const float2 before = to[i];
                    s.x += before.x;
                    s.y += before.y;
                }
                to[i] = s;
            }
            kept_tile = g.tile;
        }
    }

    const cooperative_groups::grid_group grid = cooperative_groups::this_grid();
    auto arrived = grid.barrier_arrive();
    // What the second pass needs and no other block gives.
    const float m = (float)(a.pixels * a.per);
    uint32_t next = resident ? resident - 1 : 0;                // the batch that `ahead` is at
    ahead.rewind(a, p, run, step, all, next);
    slot = (all - 1) % p.ring;
    to_slot = next % p.ring;
    grid.barrier_wait(std::move(arrived));

    for (uint32_t u = run.last;; --u) {
        if (u != run.last) {
            t = tile_of<V, L>(a, p, p.tiles == 1 ? 0 : u / (uint32_t)a.n);
            g = segment_of<V>(a, p, run, u, t);
            if (g.cnt) {
                lanes.load(a, g.c);
                lanes.stats(a, p, g.n, g.c);
                lanes.scale(lanes.w, lanes.w);
            }
            __syncthreads();  // sum of the segment before is read no more
        }
        GroupGrad<T, V, L> gg;
        join_runs<V>(a, p, t, g.n, slots, part, sum, [&](float2 v, float, uint32_t, float& s1, float& s2) {
            s1 += v.x;
            s2 += v.y;
        });
        if (g.cnt) gg.take(a, p, t, g.c, sum, m, lanes);
        uint64_t at = g.at + (g.iters - 1) / R * R * step;
        const auto give = [&](const Pack<T, V>* px, const Pack<T, V>* in, uint64_t where, bool cut_short) {
            float fx[V], fv[V];
            Pack<T, V> pv = read_vector<T, V, S>(in, where);
            read_vector<T, V, S>(px, where).get(fx);
            if (drops<DROP>(a) && (S || batch < resident)) drop_packed<S>(a.drop, dstep, where, pv);
            pv.get(fv);
            if (S && cut_short) {
                cut<V>(fx, p.tail);
                cut<V>(fv, p.tail);
            }
            if (drops<DROP>(a)) mul_v<V>(fv, fv, scale);
            lanes.grads(act_of<ACT>(a), fx, fv);
            gg.apply(lanes, fx, fv);
            Pack<T, V> o;
            o.set(fx);
            return o;
        };
        for (uint32_t i0 = (g.iters - 1) / R * R;; i0 -= R) {
            --batch;
            copy_wait<F - 1>();
            const Pack<T, V>* have = ring + slot * 2 * R * E * threads;
            if constexpr (S) {
#pragma unroll
                for (int j = 0; j < R; ++j) {  // all threads: neighbours exchange what they store
                    const uint64_t where = at + j * step;
                    const bool ok = i0 + j < g.cnt;
                    Pack<T, V> o{};
                    const bool cut_short = i0 + j + 1 == g.tail;
                    if (ok) o = give(have + 2 * j * E * threads, have + (2 * j + 1) * E * threads, where, cut_short);
                    store_shifted<T, V>((T*)a.out, where, o, ok, cut_short ? p.tail : V);
                }
            } else if (i0 + R <= g.cnt) {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    give(have + 2 * j * threads, have + (2 * j + 1) * threads, at + j * step, false).store((T*)a.out + at + j * step);
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (i0 + j < g.cnt)
                        give(have + 2 * j * threads, have + (2 * j + 1) * threads, at + j * step, false).store((T*)a.out + at + j * step);
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
    if (wanted) {
        for (uint32_t ch = block_id() * (threads / 32) + tid / 32; ch < a.c; ch += gridDim.x * gridDim.y * (threads / 32)) {
            const uint32_t tile = p.tiles == 1 ? 0 : ch / tile_c, units = (uint32_t)a.n;
            uint32_t b0, b1, none;
            runs_of_unit(p, tile * units, b0, none);
            runs_of_unit(p, (tile + 1) * units - 1, none, b1);
            join_channel<T>(a, ch, chans + (uint64_t)(b0 + tile) * tile_c + (ch - tile * tile_c), b1 - b0 + 1, tile_c);
        }
    }
}

}  // namespace norm
}  // namespace bsx
