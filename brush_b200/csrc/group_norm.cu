// group_norm.cu - group norm with an activation and dropout on channels-last tensors.
//
// Forward, for sample n and group g of Cg = C / groups channels (M = pixels Cg values):
//   mean = sum x / M, var = sum (x - mean)^2 / M, rstd = 1 / sqrt(var + eps)
//   z = gamma (x - mean) rstd + beta,  out = drop(z s(w(z)))
// with the gate s the logistic function (w = z: silu; w = 2 sqrt(2/pi) (z + 0.044715 z^3):
// the tanh form of gelu, because (1 + tanh(t)) / 2 = s(2t)) or 1 (no activation).
// Backward, with xh = (x - mean) rstd, dz = drop(v_out) d out / d z:
//   A_c = sum_pixels dz, B_c = sum_pixels dz xh          per sample and channel
//   v_bias = sum_n A, v_weight = sum_n B
//   v_x = rstd (gamma dz - (sum_g gamma A + xh sum_g gamma B) / M)
#include <new>

#include "dropout.cuh"
#include "elem.cuh"

namespace bsx {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
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

template <class T>
__device__ __forceinline__ float param(const void* p, int f32, uint32_t c, float without) {
    if (!p) return without;
    return f32 ? __ldg((const float*)p + c) : to_f(((const T*)p)[c]);
}

// The gate of the activation and d(z gate)/dz.
template <int ACT>
__device__ __forceinline__ float gate(float z) {
    if (ACT == BSX_ACT_NONE) return 1.0f;
    float w = z;
    if (ACT == BSX_ACT_GELU_TANH) w = 1.5957691216057308f * z * (1.0f + 0.044715f * z * z);
    return 1.0f / (1.0f + expf(-w));
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if (ACT == BSX_ACT_NONE) return 1.0f;
    const float s = gate<ACT>(z);
    float dw = 1.0f;
    if (ACT == BSX_ACT_GELU_TANH) dw = 1.5957691216057308f * (1.0f + 3.0f * 0.044715f * z * z);
    return s + z * s * (1.0f - s) * dw;
}

__device__ __forceinline__ float block_sum(float v, float* s) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) t += s[i];
    return t;
}

// One block per (sample, group): mean, then the squares of the deviations.
template <class T>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const NormArgs a) {
    __shared__ float s[kThreads / 32];
    const uint64_t unit = blockIdx.x, n = unit / a.groups;
    const uint32_t g = (uint32_t)(unit % a.groups);
    const T* x = (const T*)a.x + n * a.pixels * a.c + (uint64_t)g * a.per;
    const uint64_t m = a.pixels * a.per;
    float sum = 0.0f;
    for (uint64_t i = threadIdx.x; i < m; i += kThreads) sum += to_f(x[i / a.per * a.c + i % a.per]);
    const float mean = block_sum(sum, s) / (float)m;
    float sq = 0.0f;
    for (uint64_t i = threadIdx.x; i < m; i += kThreads) {
        const float d = to_f(x[i / a.per * a.c + i % a.per]) - mean;
        sq += d * d;
    }
    sq = block_sum(sq, s);
    if (threadIdx.x == 0) {
        a.mean[unit] = mean;
        a.rstd[unit] = 1.0f / sqrtf(sq / (float)m + a.eps);
    }
}

// One thread per eight consecutive elements.
template <class T, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const NormArgs a) {
    const uint64_t count = a.n * a.pixels * a.c, blocks = (count + 7) / 8;
    const uint32_t step = DROP ? drop_step(a.drop) : 0u;
    for (uint64_t b = (uint64_t)blockIdx.x * kThreads + threadIdx.x; b < blocks; b += (uint64_t)gridDim.x * kThreads) {
        const uint32_t keep = DROP ? keep8(a.drop, step, b) : 0xffu;
        for (int j = 0; j < 8; ++j) {
            const uint64_t i = b * 8 + j;
            if (i >= count) break;
            const uint32_t c = (uint32_t)(i % a.c);
            const uint64_t unit = i / a.c / a.pixels * a.groups + c / a.per;
            const float xh = (to_f(((const T*)a.x)[i]) - a.mean[unit]) * a.rstd[unit];
            const float z = xh * param<T>(a.weight, a.param_f32, c, 1.0f) + param<T>(a.bias, a.param_f32, c, 0.0f);
            float y = z * gate<ACT>(z);
            if (DROP) y = keep >> j & 1u ? y * a.drop.scale : 0.0f;
            ((T*)a.out)[i] = from_f<T>(y);
        }
    }
}

template <class T, int ACT, bool DROP>
__device__ __forceinline__ float grad_z(const NormArgs& a, uint64_t i, uint32_t c, float xh, bool keep) {
    const float z = xh * param<T>(a.weight, a.param_f32, c, 1.0f) + param<T>(a.bias, a.param_f32, c, 0.0f);
    const float v = to_f(((const T*)a.v)[i]) * act_grad<ACT>(z);
    return DROP ? (keep ? v * a.drop.scale : 0.0f) : v;
}

// One block per (sample, channel): A and B, at ws[(n C + c) 2].
template <class T, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) norm_sums_kernel(const NormArgs a) {
    __shared__ float s[kThreads / 32];
    const uint64_t n = blockIdx.x / a.c;
    const uint32_t c = blockIdx.x % a.c, step = DROP ? drop_step(a.drop) : 0u;
    const uint64_t unit = n * a.groups + c / a.per;
    const float mean = a.mean[unit], rstd = a.rstd[unit];
    float sa = 0.0f, sb = 0.0f;
    for (uint64_t p = threadIdx.x; p < a.pixels; p += kThreads) {
        const uint64_t i = (n * a.pixels + p) * a.c + c;
        const bool keep = !DROP || (keep8(a.drop, step, i / 8) >> (i & 7) & 1u);
        const float xh = (to_f(((const T*)a.x)[i]) - mean) * rstd;
        const float dz = grad_z<T, ACT, DROP>(a, i, c, xh, keep);
        sa += dz;
        sb += dz * xh;
    }
    sa = block_sum(sa, s);
    sb = block_sum(sb, s);
    if (threadIdx.x == 0) {
        a.ws[(uint64_t)blockIdx.x * 2] = sa;
        a.ws[(uint64_t)blockIdx.x * 2 + 1] = sb;
    }
}

// Parameter gradients over the samples, and the group sums at ws[2 N C + unit 2].
template <class T>
__global__ void __launch_bounds__(kThreads) norm_join_kernel(const NormArgs a) {
    const uint64_t units = a.n * a.groups;
    const uint64_t t = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (t < a.c) {
        float sa = 0.0f, sb = 0.0f;
        for (uint64_t n = 0; n < a.n; ++n) {
            sa += a.ws[(n * a.c + t) * 2];
            sb += a.ws[(n * a.c + t) * 2 + 1];
        }
        if (a.v_bias) {
            if (a.param_f32) ((float*)a.v_bias)[t] = sa;
            else ((T*)a.v_bias)[t] = from_f<T>(sa);
        }
        if (a.v_weight) {
            if (a.param_f32) ((float*)a.v_weight)[t] = sb;
            else ((T*)a.v_weight)[t] = from_f<T>(sb);
        }
    }
    if (t < units) {
        const uint64_t n = t / a.groups;
        const uint32_t g = (uint32_t)(t % a.groups);
        float s1 = 0.0f, s2 = 0.0f;
        for (uint32_t c = g * a.per; c < (g + 1) * a.per; ++c) {
            const float w = param<T>(a.weight, a.param_f32, c, 1.0f);
            s1 += w * a.ws[(n * a.c + c) * 2];
            s2 += w * a.ws[(n * a.c + c) * 2 + 1];
        }
        const float m = (float)(a.pixels * a.per);
        float* to = a.ws + a.n * a.c * 2 + t * 2;
        to[0] = s1 / m;
        to[1] = s2 / m;
    }
}

template <class T, int ACT, bool DROP>
__global__ void __launch_bounds__(kThreads) norm_grad_kernel(const NormArgs a) {
    const uint64_t count = a.n * a.pixels * a.c, blocks = (count + 7) / 8;
    const uint32_t step = DROP ? drop_step(a.drop) : 0u;
    const float* sums = a.ws + a.n * a.c * 2;
    for (uint64_t b = (uint64_t)blockIdx.x * kThreads + threadIdx.x; b < blocks; b += (uint64_t)gridDim.x * kThreads) {
        const uint32_t keep = DROP ? keep8(a.drop, step, b) : 0xffu;
        for (int j = 0; j < 8; ++j) {
            const uint64_t i = b * 8 + j;
            if (i >= count) break;
            const uint32_t c = (uint32_t)(i % a.c);
            const uint64_t unit = i / a.c / a.pixels * a.groups + c / a.per;
            const float rstd = a.rstd[unit], xh = (to_f(((const T*)a.x)[i]) - a.mean[unit]) * rstd;
            const float dz = grad_z<T, ACT, DROP>(a, i, c, xh, keep >> j & 1u);
            const float w = param<T>(a.weight, a.param_f32, c, 1.0f);
            ((T*)a.out)[i] = from_f<T>(rstd * (w * dz - (sums[unit * 2] + xh * sums[unit * 2 + 1])));
        }
    }
}

uint32_t grid_for(uint64_t threads) {
    const uint64_t b = (threads + kThreads - 1) / kThreads;
    return (uint32_t)(b < 148 * 8 ? b : 148 * 8);
}

template <class T, int ACT, bool DROP>
bsx_status forward(bsx_ctx* ctx, const NormArgs& a, cudaStream_t st) {
    prof_begin_on(ctx, st);
    norm_stats_kernel<T><<<(uint32_t)(a.n * a.groups), kThreads, 0, st>>>(a);
    bsx_status s = post_launch_on(ctx, "norm_stats_kernel", st);
    if (s != BSX_OK) return s;
    prof_begin_on(ctx, st);
    norm_apply_kernel<T, ACT, DROP><<<grid_for((a.n * a.pixels * a.c + 7) / 8), kThreads, 0, st>>>(a);
    return post_launch_on(ctx, "norm_apply_kernel", st);
}

template <class T, int ACT, bool DROP>
bsx_status backward(bsx_ctx* ctx, const NormArgs& a, cudaStream_t st) {
    prof_begin_on(ctx, st);
    norm_sums_kernel<T, ACT, DROP><<<(uint32_t)(a.n * a.c), kThreads, 0, st>>>(a);
    bsx_status s = post_launch_on(ctx, "norm_sums_kernel", st);
    if (s != BSX_OK) return s;
    const uint64_t t = a.n * a.groups > a.c ? a.n * a.groups : a.c;
    prof_begin_on(ctx, st);
    norm_join_kernel<T><<<(uint32_t)((t + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
    s = post_launch_on(ctx, "norm_join_kernel", st);
    if (s != BSX_OK) return s;
    prof_begin_on(ctx, st);
    norm_grad_kernel<T, ACT, DROP><<<grid_for((a.n * a.pixels * a.c + 7) / 8), kThreads, 0, st>>>(a);
    return post_launch_on(ctx, "norm_grad_kernel", st);
}

template <class T, int ACT>
bsx_status by_drop(bsx_ctx* ctx, const NormArgs& a, bool drop, bool bwd, cudaStream_t st) {
    if (bwd) return drop ? backward<T, ACT, true>(ctx, a, st) : backward<T, ACT, false>(ctx, a, st);
    return drop ? forward<T, ACT, true>(ctx, a, st) : forward<T, ACT, false>(ctx, a, st);
}

template <class T>
bsx_status by_act(bsx_ctx* ctx, const NormArgs& a, int act, bool drop, bool bwd, cudaStream_t st) {
    if (act == BSX_ACT_NONE) return by_drop<T, BSX_ACT_NONE>(ctx, a, drop, bwd, st);
    if (act == BSX_ACT_SILU) return by_drop<T, BSX_ACT_SILU>(ctx, a, drop, bwd, st);
    return by_drop<T, BSX_ACT_GELU_TANH>(ctx, a, drop, bwd, st);
}

// Sizes the kernels index with: blocks fit a grid, products fit 64 bits.
const char* bad_sizes(uint64_t n, uint64_t pixels, uint32_t c, uint32_t groups) {
    if (c == 0 || groups == 0 || c % groups) return "channels must be a positive multiple of groups";
    const uint64_t limit = 0x7fffffffu;
    if (n > limit / c) return "samples x channels must stay below 2^31";
    if (pixels && n && pixels > (UINT64_MAX >> 4) / ((uint64_t)n * c)) return "too many elements";
    return nullptr;
}

uint64_t workspace_floats(uint64_t n, uint64_t pixels, uint32_t c, uint32_t groups, bool bwd) {
    (void)pixels;
    return bwd ? 2 * n * c + 2 * n * groups : 4;
}

bsx_status run(bsx_ctx* ctx, NormArgs a, int32_t dtype, const bsx_group_norm_cfg* cfg, void* ws, uint64_t ws_bytes,
               bool bwd, void* stream) {
    if (!ctx || !cfg) return BSX_ERR_INVALID_ARG;
    try {
        std::lock_guard<std::mutex> lock(ctx->op_mutex);
        auto bad = [&](const char* why) { return fail(ctx, BSX_ERR_INVALID_ARG, why); };
        if (dtype < BSX_F32 || dtype > BSX_F16) return bad("unknown element type");
        if (cfg->param_dtype != BSX_F32 && cfg->param_dtype != dtype)
            return bad("weight and bias must be float or of the tensor's type");
        if (cfg->activation < BSX_ACT_NONE || cfg->activation > BSX_ACT_GELU_TANH) return bad("unknown activation");
        if (!(cfg->eps >= 0.0f)) return bad("eps must not be negative");
        if (const char* why = bad_sizes(a.n, a.pixels, a.c, cfg->groups)) return fail(ctx, BSX_ERR_SHAPE, why);
        a.groups = cfg->groups;
        a.per = a.c / cfg->groups;
        a.eps = cfg->eps;
        a.param_f32 = cfg->param_dtype == BSX_F32;
        a.ws = (float*)ws;
        const bool drop = cfg->dropout != nullptr;
        if (drop) {
            if (const char* why = drop_args(cfg->dropout, &a.drop)) return bad(why);
            if (cfg->dropout->share != 1) return bad("dropout in a group norm draws for each element (share 1)");
        }
        const uintptr_t size = dtype == BSX_F32 ? 4 : 2, psize = a.param_f32 ? 4 : 2;
        if (((uintptr_t)a.x | (uintptr_t)a.v | (uintptr_t)a.out) % size ||
            ((uintptr_t)a.weight | (uintptr_t)a.bias | (uintptr_t)a.v_weight | (uintptr_t)a.v_bias) % psize ||
            ((uintptr_t)a.mean | (uintptr_t)a.rstd) % 4 || (uintptr_t)ws % 16)
            return bad("tensors must be aligned to their elements, the workspace to 16 bytes");
        if (a.pixels == 0) return fail(ctx, BSX_ERR_SHAPE, "a sample must have at least one pixel");
        if (a.n && (!a.x || !a.out || (bwd && !a.v))) return bad("null tensor");
        if (a.n && (!a.mean || !a.rstd)) return bad("null mean or rstd");
        const uint64_t need = workspace_floats(a.n, a.pixels, a.c, a.groups, bwd) * 4;
        if (ws_bytes < need || (need && !ws)) return fail(ctx, BSX_ERR_CAPACITY, "the workspace is too small");
        DeviceScope on(ctx->device);
        const cudaStream_t st = (cudaStream_t)stream;
        if (a.n == 0) {  // no samples: parameter gradients of nothing are 0
            for (void* to : {a.v_weight, a.v_bias})
                if (bwd && to) {
                    const bsx_status s = check_cuda(ctx, cudaMemsetAsync(to, 0, a.c * psize, st), "memset");
                    if (s != BSX_OK) return s;
                }
            return BSX_OK;
        }
        if (dtype == BSX_F32) return by_act<float>(ctx, a, cfg->activation, drop, bwd, st);
        if (dtype == BSX_BF16) return by_act<__nv_bfloat16>(ctx, a, cfg->activation, drop, bwd, st);
        return by_act<__half>(ctx, a, cfg->activation, drop, bwd, st);
    } catch (...) {
        return BSX_ERR_CAPACITY;  // host allocation failed while writing the error text
    }
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" {

bsx_status bsx_group_norm_workspace(uint64_t n, uint64_t pixels, uint32_t channels, uint32_t groups, int32_t backward,
                                    uint64_t* bytes) {
    if (!bytes) return BSX_ERR_INVALID_ARG;
    *bytes = 0;
    if (bad_sizes(n, pixels, channels, groups)) return BSX_ERR_SHAPE;
    *bytes = workspace_floats(n, pixels, channels, groups, backward != 0) * 4;
    return BSX_OK;
}

bsx_status bsx_group_norm_fwd(bsx_ctx* ctx, const void* d_x, const void* d_weight, const void* d_bias, uint64_t n,
                              uint64_t pixels, uint32_t channels, int32_t dtype, const bsx_group_norm_cfg* cfg,
                              void* d_out, float* d_mean, float* d_rstd, void* d_workspace, uint64_t workspace_bytes,
                              void* stream) {
    NormArgs a{};
    a.x = d_x;
    a.weight = d_weight;
    a.bias = d_bias;
    a.out = d_out;
    a.mean = d_mean;
    a.rstd = d_rstd;
    a.n = n;
    a.pixels = pixels;
    a.c = channels;
    return run(ctx, a, dtype, cfg, d_workspace, workspace_bytes, false, stream);
}

bsx_status bsx_group_norm_bwd(bsx_ctx* ctx, const void* d_v_out, const void* d_x, const void* d_weight,
                              const void* d_bias, const float* d_mean, const float* d_rstd, uint64_t n, uint64_t pixels,
                              uint32_t channels, int32_t dtype, const bsx_group_norm_cfg* cfg, void* d_v_x,
                              void* d_v_weight, void* d_v_bias, void* d_workspace, uint64_t workspace_bytes,
                              void* stream) {
    NormArgs a{};
    a.x = d_x;
    a.v = d_v_out;
    a.weight = d_weight;
    a.bias = d_bias;
    a.out = d_v_x;
    a.mean = const_cast<float*>(d_mean);
    a.rstd = const_cast<float*>(d_rstd);
    a.v_weight = d_v_weight;
    a.v_bias = d_v_bias;
    a.n = n;
    a.pixels = pixels;
    a.c = channels;
    return run(ctx, a, dtype, cfg, d_workspace, workspace_bytes, true, stream);
}

}  // extern "C"
