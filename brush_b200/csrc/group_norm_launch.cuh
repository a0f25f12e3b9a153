// group_norm_launch.cuh - the group-norm kernels of one element type and their launches.
#pragma once

#include <atomic>

#include "group_norm_bwd.cuh"
#include "group_norm_fwd.cuh"

namespace bsx {
namespace norm {

constexpr uint32_t kSharedMost = 227 * 1024;

// SMs of a device, and whether a kernel may take all of its shared memory (set once a kernel and device).
inline int sm_count(int device) {
    static std::atomic<int> known[64];
    if (device < 0 || device >= 64) return 1;
    int n = known[device].load();
    if (!n && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess) known[device].store(n);
    return n > 0 ? n : 1;
}
template <class K>
cudaError_t prepare(K kernel, std::atomic<uint64_t>& done, int device) {
    if (device >= 0 && device < 64 && done.load() >> device & 1) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedMost);
    if (e == cudaSuccess && device >= 0 && device < 64) done.fetch_or(1ull << device);
    return e;
}

template <class K>
cudaError_t cooperative(K kernel, const Args& a, const Plan& p, dim3 blocks, uint32_t bytes, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks;
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p, a);
}

template <class T, int V, int L, int ACT, int DROP, bool BWD, bool S = false>
cudaError_t launch_one(const Call& c) {
    const Args& a = *c.a;
    Plan& p = *c.p;
    const int sms = sm_count(c.device);
    const uint32_t sums = 8 * (p.gl + kThreads / 32);  // sum, warp_sum
    if constexpr (!BWD && !S) if (p.small) {
        static std::atomic<uint64_t> done{0};
        auto k = small_fwd_kernel<T, V, L, ACT, DROP>;
        if (cudaError_t e = prepare(k, done, c.device)) return e;
        k<<<p.blocks, p.threads, sums + 16 + 4 * (p.gl + places<L>(p.threads)), c.stream>>>(p, a);
        return cudaSuccess;
    }
    if constexpr (BWD && !S) if (p.small) {
        static std::atomic<uint64_t> done{0};
        auto k = small_bwd_kernel<T, V, L, ACT, DROP>;
        if (cudaError_t e = prepare(k, done, c.device)) return e;
        const uint32_t bytes = sums + 16 + 8 * places<V>(p.threads);
        // blocks that fit an SM with these threads and bytes; the last answer is kept, a query costs as much as a launch
        static std::atomic<uint64_t> known{0};
        int per_sm = 1;
        if (p.blocks > (uint32_t)sms) {
            const uint64_t key = (uint64_t)p.threads << 40 | (uint64_t)bytes << 16, got = known.load();
            if (got >> 16 << 16 == key) {
                per_sm = (int)(got & 0xffff);
            } else {
                if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, (int)p.threads, bytes)) return e;
                known.store(key | (uint64_t)per_sm);
            }
        }
        const uint32_t most = (uint32_t)(sms * per_sm) < kMaxBlocks ? (uint32_t)(sms * per_sm) : kMaxBlocks;
        return cooperative(k, a, p, p.blocks < most ? p.blocks : most / p.tiles * p.tiles, bytes, c.stream);
    }
    const uint32_t tile_c = p.tiles == 1 ? a.c : p.cols * V;
    const uint32_t head = 32 + sums + (BWD ? 8 * (tile_c + places<V>(p.threads)) : 4 * p.gl + 8 * places<L>(p.threads));
    const uint32_t row = p.threads * (uint32_t)sizeof(Pack<T, V>) * (BWD ? 2 : 1) * (S ? 2 : 1);  // a single 16-bit element takes a word
    // Where units are few, each has blocks of its own, so that no block sums and joins twice; where that would
    // leave more than a tenth of the SMs idle, runs cross units.
    const uint32_t units = (uint32_t)a.n * p.tiles, total = p.rows * units;
    uint32_t blocks = total < (uint32_t)sms ? total : (uint32_t)sms;
    p.per_unit = blocks / units;
    if (p.per_unit > 0 && p.per_unit * units * 10 >= blocks * 9) {
        p.each = p.rows / p.per_unit;
        p.more = p.rows % p.per_unit;
        p.per_block = p.each + 1;
        blocks = p.per_unit * units;
    } else {
        p.per_unit = 0;
        p.per_block = (total + blocks - 1) / blocks;
        blocks = (total + p.per_block - 1) / p.per_block;
    }
    constexpr uint32_t rows = rows_of_batch(BWD, S);
    const uint32_t batch = rows * row;
    // the longest run's batches: its rows, and a cut batch at each end of a unit
    const uint32_t longest = p.per_block / rows + 1 + (p.per_unit ? 0 : p.per_block / p.rows + 1);
    p.ring = (kSharedMost - 16 - head) / batch;
    if (p.ring > longest) p.ring = longest;
    const uint32_t bytes = head + 16 + p.ring * batch;
    const dim3 grid = p.per_unit ? dim3(p.per_unit, units) : dim3(blocks);
    static std::atomic<uint64_t> done{0};
    const auto k = [] {
        if constexpr (BWD) return large_bwd_kernel<T, V, L, ACT, DROP, S>;
        else return large_fwd_kernel<T, V, L, ACT, DROP, S>;
    }();
    if (cudaError_t e = prepare(k, done, c.device)) return e;
    return cooperative(k, a, p, grid, bytes, c.stream);
}

template <class T, int V, int L, bool BWD>
cudaError_t by_act(const Call& c) {
    const bool drop = c.a->dropping;
    switch (c.a->act) {
        case BSX_ACT_NONE:
            return drop ? launch_one<T, V, L, BSX_ACT_NONE, 1, BWD>(c) : launch_one<T, V, L, BSX_ACT_NONE, 0, BWD>(c);
        case BSX_ACT_SILU:
            return drop ? launch_one<T, V, L, BSX_ACT_SILU, 1, BWD>(c) : launch_one<T, V, L, BSX_ACT_SILU, 0, BWD>(c);
    }
    return drop ? launch_one<T, V, L, BSX_ACT_GELU_TANH, 1, BWD>(c) : launch_one<T, V, L, BSX_ACT_GELU_TANH, 0, BWD>(c);
}

template <class T, bool BWD>
cudaError_t launch(const Call& c) {
    constexpr int M = 16 / (int)sizeof(T);
    if constexpr (M == 8) if (c.p->shifted) return launch_one<T, M, M, kAny, kAny, BWD, true>(c);
    if (c.p->v == M) {
        if (c.items == 1) return by_act<T, M, 1, BWD>(c);
        if (c.items == 2) return by_act<T, M, 2, BWD>(c);
        if (M == 4 || c.items == 4) return launch_one<T, M, 4, kAny, kAny, BWD>(c);
        return launch_one<T, M, M, kAny, kAny, BWD>(c);
    }
    if (c.p->v == 2) return launch_one<T, 2, 2, kAny, kAny, BWD>(c);
    return launch_one<T, 1, 1, kAny, kAny, BWD>(c);
}
template <class T>
cudaError_t launch_fwd(const Call& c) {
    return launch<T, false>(c);
}
template <class T>
cudaError_t launch_bwd(const Call& c) {
    return launch<T, true>(c);
}

}  // namespace norm
}  // namespace bsx
