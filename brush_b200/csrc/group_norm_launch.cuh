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
cudaError_t cooperative(K kernel, const Args& a, const Plan& p, uint32_t blocks, uint32_t bytes, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, p);
}

template <class T, int V, int L, int ACT, bool DROP>
cudaError_t launch_one(const Call& c) {
    const Args& a = *c.a;
    Plan& p = *c.p;
    static std::atomic<uint64_t> done_small{0}, done_large{0};
    const int sms = sm_count(c.device);
    if (p.small) {
        if (!c.bwd) {
            const uint32_t bytes = (sums_floats(p.threads, L, p.gl, false) + p.gl) * 4;
            auto k = small_fwd_kernel<T, V, L, ACT, DROP>;
            if (cudaError_t e = prepare(k, done_small, c.device)) return e;
            k<<<p.blocks, p.threads, bytes, c.stream>>>(a, p);
            return cudaSuccess;
        }
        const uint32_t bytes = sums_floats(p.threads, V, p.gl, true) * 4;
        auto k = small_bwd_kernel<T, V, L, ACT, DROP>;
        static std::atomic<uint64_t> done{0};
        if (cudaError_t e = prepare(k, done, c.device)) return e;
        int per_sm = 1;
        if (p.blocks > (uint32_t)sms) {
            if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, (int)p.threads, bytes)) return e;
        }
        uint32_t most = (uint32_t)(sms * per_sm);
        if (most > kMaxBlocks) most = kMaxBlocks;
        uint32_t blocks = p.blocks < most ? p.blocks : most / p.tiles * p.tiles;
        return cooperative(k, a, p, blocks, bytes, c.stream);
    }
    const uint32_t head = (sums_floats(p.threads, c.bwd ? V : L, p.gl, c.bwd) * 4 + 15) / 16 * 16;
    const uint32_t slot = p.threads * (uint32_t)sizeof(Pack<T, V>) * (c.bwd ? 2 : 1);  // a single 16-bit element takes a word
    p.keep = (kSharedMost - 16 - head) / slot;
    const uint64_t total = p.rows * a.n * p.tiles;
    uint64_t blocks = (total + p.k - 1) / p.k;
    if (blocks > (uint64_t)sms) blocks = sms;
    p.per_block = ((total + blocks - 1) / blocks + p.k - 1) / p.k * p.k;
    blocks = (total + p.per_block - 1) / p.per_block;
    // no more shared memory than the longest run can use
    const uint64_t iters = (p.per_block + p.k - 1) / p.k + p.per_block / p.rows + 2;
    if (p.keep > iters) p.keep = (uint32_t)iters;
    const uint32_t bytes = head + 16 + p.keep * slot;
    if (c.bwd) {
        auto k = large_bwd_kernel<T, V, L, ACT, DROP>;
        static std::atomic<uint64_t> done{0};
        if (cudaError_t e = prepare(k, done, c.device)) return e;
        return cooperative(k, a, p, (uint32_t)blocks, bytes, c.stream);
    }
    auto k = large_fwd_kernel<T, V, L, ACT, DROP>;
    if (cudaError_t e = prepare(k, done_large, c.device)) return e;
    return cooperative(k, a, p, (uint32_t)blocks, bytes, c.stream);
}

template <class T, int V, int L>
cudaError_t by_act(const Call& c) {
    if (c.act == BSX_ACT_NONE)
        return c.drop ? launch_one<T, V, L, BSX_ACT_NONE, true>(c) : launch_one<T, V, L, BSX_ACT_NONE, false>(c);
    if (c.act == BSX_ACT_SILU)
        return c.drop ? launch_one<T, V, L, BSX_ACT_SILU, true>(c) : launch_one<T, V, L, BSX_ACT_SILU, false>(c);
    return c.drop ? launch_one<T, V, L, BSX_ACT_GELU_TANH, true>(c) : launch_one<T, V, L, BSX_ACT_GELU_TANH, false>(c);
}

template <class T>
cudaError_t launch(const Call& c) {
    constexpr int kMost = 16 / (int)sizeof(T);
    if (c.p->v == kMost) return c.whole ? by_act<T, kMost, 1>(c) : by_act<T, kMost, kMost>(c);
    if constexpr (sizeof(T) == 2)
        if (c.p->v == 2) return by_act<T, 2, 2>(c);
    return by_act<T, 1, 1>(c);
}

}  // namespace norm
}  // namespace bsx
