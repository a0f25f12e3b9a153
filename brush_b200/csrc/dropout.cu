// dropout.cu - dropout with a counter-based mask that is never stored.
//
// Forward y = residual + x m / (1 - p), backward v_x = v_y m / (1 - p), with m drawn again
// from (seed, step, draw index) each time (dropout.cuh). Products and sums are formed in
// 32 bits and rounded once. A dropped element is a select, not a product with zero, so
// infinities and NaN in dropped places leave nothing behind.
#include <cmath>
#include <new>

#include "dropout.cuh"
#include "elem.cuh"

namespace bsx {

const char* drop_args(const bsx_dropout_cfg* cfg, DropArgs* out) {
    if (!(cfg->p >= 0.0 && cfg->p <= 1.0)) return "dropout p must lie in [0, 1]";
    if ((uintptr_t)cfg->d_step % 4) return "the dropout step must be 4-byte aligned";
    const uint64_t t = (uint64_t)std::nearbyint(cfg->p * 4294967296.0);  // half to even; 2^32 for p = 1
    out->k0 = (uint32_t)cfg->seed;
    out->k1 = (uint32_t)(cfg->seed >> 32);
    out->step = cfg->step;
    out->d_step = cfg->d_step;
    out->t_hi = (uint32_t)(t >> 16);
    out->t_lo = (uint32_t)(t & 0xffff);
    out->scale = cfg->p < 1.0 ? (float)(1.0 / (1.0 - cfg->p)) : 0.0f;
    return nullptr;
}

namespace {

constexpr int kThreads = 256;

// One thread per eight consecutive elements.
template <class T, bool RES>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out, uint64_t n, uint64_t share,
                   const DropArgs d) {
    const uint32_t step = drop_step(d);
    const uint64_t blocks = (n + 7) / 8;
    for (uint64_t b = (uint64_t)blockIdx.x * kThreads + threadIdx.x; b < blocks; b += (uint64_t)gridDim.x * kThreads) {
        uint64_t have = UINT64_MAX;
        uint32_t keep = 0;
        for (int j = 0; j < 8; ++j) {
            const uint64_t i = b * 8 + j;
            if (i >= n) break;
            const uint64_t m = i / share;
            if (m / 8 != have) {
                have = m / 8;
                keep = keep8(d, step, have);
            }
            float v = keep >> (m & 7) & 1u ? to_f(x[i]) * d.scale : 0.0f;
            if (RES) v += to_f(res[i]);
            out[i] = from_f<T>(v);
        }
    }
}

template <class T>
void launch(const void* x, const void* res, void* out, uint64_t n, uint64_t share, const DropArgs& d, cudaStream_t st) {
    const uint64_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
    const uint32_t grid = (uint32_t)(blocks < 148 * 8 ? blocks : 148 * 8);
    if (res)
        dropout_kernel<T, true><<<grid, kThreads, 0, st>>>((const T*)x, (const T*)res, (T*)out, n, share, d);
    else
        dropout_kernel<T, false><<<grid, kThreads, 0, st>>>((const T*)x, nullptr, (T*)out, n, share, d);
}

bsx_status run(bsx_ctx* ctx, const char* name, const void* x, const void* res, uint64_t n, int32_t dtype,
               const bsx_dropout_cfg* cfg, void* out, void* stream) {
    if (!ctx || !cfg) return BSX_ERR_INVALID_ARG;
    try {
        std::lock_guard<std::mutex> lock(ctx->op_mutex);
        DropArgs d;
        if (const char* why = drop_args(cfg, &d)) return fail(ctx, BSX_ERR_INVALID_ARG, why);
        if (cfg->share == 0) return fail(ctx, BSX_ERR_INVALID_ARG, "dropout share must be at least 1");
        if (dtype < BSX_F32 || dtype > BSX_F16) return fail(ctx, BSX_ERR_INVALID_ARG, "unknown element type");
        if (n == 0) return BSX_OK;
        if (n > (UINT64_MAX >> 4)) return fail(ctx, BSX_ERR_CAPACITY, "too many elements");
        if (!x || !out) return fail(ctx, BSX_ERR_INVALID_ARG, "null tensor");
        const uintptr_t size = dtype == BSX_F32 ? 4 : 2;
        if (((uintptr_t)x | (uintptr_t)out | (uintptr_t)res) % size)
            return fail(ctx, BSX_ERR_INVALID_ARG, "tensors must be aligned to their elements");
        DeviceScope on(ctx->device);
        const cudaStream_t st = (cudaStream_t)stream;
        prof_begin_on(ctx, st);
        if (dtype == BSX_F32) launch<float>(x, res, out, n, cfg->share, d, st);
        else if (dtype == BSX_BF16) launch<__nv_bfloat16>(x, res, out, n, cfg->share, d, st);
        else launch<__half>(x, res, out, n, cfg->share, d, st);
        return post_launch_on(ctx, name, st);
    } catch (...) {
        return BSX_ERR_CAPACITY;  // host allocation failed while writing the error text
    }
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" {

bsx_status bsx_dropout_fwd(bsx_ctx* ctx, const void* d_x, const void* d_residual, uint64_t count, int32_t dtype,
                           const bsx_dropout_cfg* cfg, void* d_out, void* stream) {
    return run(ctx, "dropout_fwd_kernel", d_x, d_residual, count, dtype, cfg, d_out, stream);
}

bsx_status bsx_dropout_bwd(bsx_ctx* ctx, const void* d_v_out, uint64_t count, int32_t dtype, const bsx_dropout_cfg* cfg,
                           void* d_v_x, void* stream) {
    return run(ctx, "dropout_bwd_kernel", d_v_out, nullptr, count, dtype, cfg, d_v_x, stream);
}

}  // extern "C"
