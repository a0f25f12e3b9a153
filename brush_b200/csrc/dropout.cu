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
    for (uint32_t r = 0; r < kRounds; ++r) {
        out->k0[r] = (uint32_t)cfg->seed + r * 0x9E3779B9u;
        out->k1[r] = (uint32_t)(cfg->seed >> 32) + r * 0xBB67AE85u;
    }
    out->step = cfg->step;
    out->d_step = cfg->d_step;
    out->t_hi = t >> 32 ? 65535u : (uint32_t)(t >> 16);  // nothing exceeds 65535 and no low halfword reaches 65536
    out->t_lo = t >> 32 ? 65536u : (uint32_t)(t & 0xffff);
    out->scale = cfg->p < 1.0 ? (float)(1.0 / (1.0 - cfg->p)) : 0.0f;
    return nullptr;
}

namespace {

constexpr int kThreads = 256;
constexpr uint64_t kMaxElements = 1ull << 42;  // the grid's limit is 2^31 blocks of 8192 elements
// Blocks of eight elements that a thread has in flight. Four fill the memory pipe with 16 warps an SM (half
// a frame, 33 M bf16 elements with a residual, 199 MB: 32.1 us against 33.9 with two and 33.4 with one); below
// the count where four a thread leave SMs without work, one.
constexpr int kMany = 4;
constexpr uint64_t kManyFrom = 148ull * 4 * kThreads * kMany;

// share > 1: the eight elements from i (a multiple of 8) belong to rows m, m + 1, ... of `share` elements: to one
// where share is a multiple of 8, to two at most from 8 on, and to five at most (share 2) below. The branches are
// the same for a whole launch.
__device__ __forceinline__ void drop_rows(const DropArgs& d, uint32_t step, uint64_t i, const Divisor& share,
                                          float (&v)[8]) {
    const uint64_t m = share.of(i);
    if (share.d % 8 == 0) {
        const bool all = keep1(d, step, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = all ? v[j] * d.scale : 0.0f;
        return;
    }
    const uint64_t rest = share.d - (i - m * share.d);  // elements of row m from i on
    uint32_t left = rest < 8 ? (uint32_t)rest : 8u, keep = keep8(d, step, m >> 3) >> (m & 7);
    if (share.d > 8) {
        if (left < 8 && (m & 7) == 7) keep |= keep8(d, step, (m >> 3) + 1) << 1;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (j < left ? keep & 1u : keep & 2u) ? v[j] * d.scale : 0.0f;
        return;
    }
    const uint32_t by = (uint32_t)share.d;
    if ((m & 7) + (7 - left) / by + 1 > 7) keep |= keep8(d, step, (m >> 3) + 1) << (8 - (m & 7));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (left == 0) {
            keep >>= 1;
            left = by;
        }
        --left;
        v[j] = keep & 1u ? v[j] * d.scale : 0.0f;
    }
}

template <bool ROWS>
__device__ __forceinline__ void drop8(const DropArgs& d, uint32_t step, uint64_t b, const Divisor& share, float (&v)[8]) {
    if (ROWS) drop_rows(d, step, b * 8, share, v);
    else drop_values<8>(d, step, b, v);
}

// A block of eight elements by single accesses: the last, partial block, and tensors that are not on 16 bytes.
template <class T, bool RES, bool ROWS>
__device__ __forceinline__ void single8(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out,
                                        uint64_t b, uint64_t n, const Divisor& share, const DropArgs& d, uint32_t step) {
    const uint64_t i = b * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? to_f(x[i + j]) : 0.0f;
    drop8<ROWS>(d, step, b, share, v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < n) out[i + j] = from_f<T>(RES ? v[j] + to_f(res[i + j]) : v[j]);
}

// One thread per block of eight elements, U blocks a thread, kThreads apart. Memory bounds it: a million rows of 48
// floats, a draw a row, 384 MB in 60.6 us (6.3 TB/s, 97 % of the measured copy rate); 33 M bf16 elements with a
// residual, 199 MB in 32.3 us (94 %). Without a residual 16-bit elements have 14 instructions each (seven rounds, the
// comparisons and conversions): 14.4 M f16 elements, 58 MB, 12.7 us (69 %). Neither memory nor issue bounds that: while
// an SM has blocks it issues 63 % of the time, but over the whole launch 47 %, since three waves of blocks begin with
// loads and end unevenly. Tried: a grid of resident blocks that loops (13.7 to
// 14.9 us there, 75 us for the rows): the loads of an iteration then wait for the iteration before.
template <class T, bool RES, bool ROWS, bool VEC, int U>
__global__ void __launch_bounds__(kThreads, 4)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out, uint64_t n,
                   const Divisor share, const DropArgs d) {
    const uint32_t step = drop_step(d);
    const uint64_t whole = n / 8, b0 = (uint64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
    if (VEC) {
        Pack<T, 8> v[U], r[U];  // packed: registers decide how many loads are in flight
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint64_t b = b0 + k * kThreads;
            if (b < whole) {
                v[k].load(x + b * 8);
                if (RES) r[k].load(res + b * 8);
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint64_t b = b0 + k * kThreads;
            if (b < whole) {
                float f[8];
                v[k].get(f);
                drop8<ROWS>(d, step, b, share, f);
                if (RES) {
                    float g[8];
                    r[k].get(g);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] += g[j];
                }
                v[k].set(f);
                v[k].store(out + b * 8);
            }
        }
        if (b0 == 0 && whole * 8 < n) single8<T, RES, ROWS>(x, res, out, whole, n, share, d, step);
    } else {
#pragma unroll 1
        for (int k = 0; k < U; ++k) {
            const uint64_t b = b0 + k * kThreads;
            if (b * 8 < n) single8<T, RES, ROWS>(x, res, out, b, n, share, d, step);
        }
    }
}

template <class T, bool RES, bool ROWS>
void launch(const T* x, const T* res, T* out, uint64_t n, const Divisor& share, const DropArgs& d, cudaStream_t st) {
    const uint64_t blocks = (n + 7) / 8;
    const bool vec = ((uintptr_t)x | (uintptr_t)res | (uintptr_t)out) % 16 == 0;
    const int u = blocks >= kManyFrom ? kMany : 1;
    const uint32_t grid = (uint32_t)((blocks + kThreads * u - 1) / (kThreads * u));
    if (vec && u > 1) dropout_kernel<T, RES, ROWS, true, kMany><<<grid, kThreads, 0, st>>>(x, res, out, n, share, d);
    else if (vec) dropout_kernel<T, RES, ROWS, true, 1><<<grid, kThreads, 0, st>>>(x, res, out, n, share, d);
    else if (u > 1) dropout_kernel<T, RES, ROWS, false, kMany><<<grid, kThreads, 0, st>>>(x, res, out, n, share, d);
    else dropout_kernel<T, RES, ROWS, false, 1><<<grid, kThreads, 0, st>>>(x, res, out, n, share, d);
}

template <class T>
void launch(const void* x, const void* res, void* out, uint64_t n, uint64_t share, const DropArgs& d, cudaStream_t st) {
    const Divisor by(share, n);
    const T *tx = (const T*)x, *tr = (const T*)res;
    if (res && share > 1) launch<T, true, true>(tx, tr, (T*)out, n, by, d, st);
    else if (res) launch<T, true, false>(tx, tr, (T*)out, n, by, d, st);
    else if (share > 1) launch<T, false, true>(tx, tr, (T*)out, n, by, d, st);
    else launch<T, false, false>(tx, tr, (T*)out, n, by, d, st);
}

bsx_status run(bsx_ctx* ctx, const char* name, const void* x, const void* res, uint64_t n, int32_t dtype,
               const bsx_dropout_cfg* cfg, void* out, void* stream) {
    if (!ctx || !cfg) return BSX_ERR_INVALID_ARG;
    try {
        DropArgs d;
        if (const char* why = drop_args(cfg, &d)) return fail(ctx, BSX_ERR_INVALID_ARG, why);
        if (cfg->share == 0) return fail(ctx, BSX_ERR_INVALID_ARG, "dropout share must be at least 1");
        if (dtype < BSX_F32 || dtype > BSX_F16) return fail(ctx, BSX_ERR_INVALID_ARG, "unknown element type");
        if (n == 0) return BSX_OK;
        if (n > kMaxElements) return fail(ctx, BSX_ERR_CAPACITY, "too many elements");
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
