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
//
// The kernels are in group_norm_fwd.cuh and group_norm_bwd.cuh; here are the checks, the cut of
// a tensor into blocks, and the entry points.
#include <numeric>

#include "group_norm.cuh"

namespace bsx {
namespace norm {
extern template cudaError_t launch_fwd<float>(const Call&);
extern template cudaError_t launch_fwd<__nv_bfloat16>(const Call&);
extern template cudaError_t launch_fwd<__half>(const Call&);
extern template cudaError_t launch_bwd<float>(const Call&);
extern template cudaError_t launch_bwd<__nv_bfloat16>(const Call&);
extern template cudaError_t launch_bwd<__half>(const Call&);
}  // namespace norm

namespace {
using namespace norm;

// Sizes the kernels index with: blocks fit a grid, products fit 64 bits.
const char* bad_sizes(uint64_t n, uint64_t pixels, uint32_t c, uint32_t groups) {
    if (c == 0 || groups == 0 || c % groups) return "channels must be a positive multiple of groups";
    const uint64_t limit = 0x7fffffffu;
    if (n > limit / c) return "samples x channels must stay below 2^31";
    if (pixels && n && pixels > (UINT64_MAX >> 4) / ((uint64_t)n * c)) return "too many elements";
    return nullptr;
}

uint32_t groups_of_tile(uint32_t c, uint32_t per, uint32_t channels, uint32_t tiles) {
    if (tiles == 1) return c / per;
    if (channels % per == 0) return channels / per;
    return (channels - 1) / per + 2;  // cut groups at both ends
}

// The cut for vectors of v elements; v divides a sample, or the vectors are shifted. False: more rows than the
// kernels count.
bool plan_for(uint64_t n, uint64_t pixels, uint32_t c, uint32_t groups, uint32_t v, bool bwd, bool shifted, Plan& p) {
    const uint32_t per = c / groups, batch = bwd ? kBatchBwd : kBatch;
    p = Plan{};
    p.v = v;
    p.elems = pixels * c;
    p.vecs = (p.elems + v - 1) / v;
    p.shifted = shifted;
    p.tail = (uint32_t)(p.elems % v);
    p.by_per = Div32::of(per, c);
    p.by_c = Div32::of(c, (uint64_t)kThreads * 8);
    const uint32_t run = c / std::gcd(c, v);  // the shortest row
    const uint64_t rows = (p.vecs + run - 1) / run;
    // Small: a block holds a (sample, tile) in registers. Tiles are whole groups and at least half a sector wide.
    const auto fits = [&](uint64_t cols) { return cols <= (uint64_t)kThreads && rows <= (kThreads / cols) * batch; };
    uint64_t cols = 0;
    if (shifted) {
    } else if (fits(run)) {
        cols = run;
    } else if (c % v == 0) {
        const uint64_t unit = std::lcm((uint64_t)per, (uint64_t)v) / v;
        if (fits(unit)) cols = unit;
        while (cols && cols + unit < run && fits(cols + unit)) cols += unit;
        if (cols * v < 16 || (run + cols - 1) / (cols ? cols : 1) > 64) cols = 0;
    }
    if (cols) {
        p.small = 1;
        p.rv = run;
        p.rows = (uint32_t)rows;
        p.cols = (uint32_t)cols;
        p.k = kThreads / p.cols < p.rows ? kThreads / p.cols : p.rows;
    } else {
        p.rv = run < (uint32_t)kThreads ? kThreads / run * run : run;
        const uint64_t wide = (p.vecs + p.rv - 1) / p.rv;
        if (wide >= 1ull << 31) return false;
        p.rows = (uint32_t)wide;
        p.cols = p.rv < (uint32_t)kThreads ? p.rv : kThreads;
        p.k = 1;
    }
    p.last = (uint32_t)(p.vecs - (uint64_t)(p.rows - 1) * p.rv);
    p.tiles = (p.rv + p.cols - 1) / p.cols;
    p.pixels = p.tiles > 1 ? 1 : p.rv * v / c;
    p.pixels_last = p.tiles > 1 ? 1 : (uint32_t)((p.elems - (uint64_t)(p.rows - 1) * p.rv * v) / c);
    p.threads = (p.k * p.cols + 31) / 32 * 32;
    p.blocks = p.small ? (uint32_t)(n * p.tiles) : 0;
    p.gl = groups_of_tile(c, per, p.cols * v, p.tiles);
    p.by_cols = Div32::of(p.cols, kThreads);
    return p.small || (uint64_t)p.rows * n * p.tiles < 1ull << 31;
}

// Floats of workspace: the partial sums that plan_for's kernels leave (group_norm_fwd.cuh, group_norm_bwd.cuh).
uint64_t workspace_of(const Plan& p, uint64_t n, uint32_t c, bool bwd) {
    if (p.small) return bwd ? 2ull * kMaxBlocks * c : 0;
    const uint64_t slots = (kMaxBlocks + (uint64_t)p.tiles * n) * p.gl;
    if (!bwd) return 2 * slots;
    return 2 * slots + 2 * (kMaxBlocks + (uint64_t)p.tiles) * (p.tiles == 1 ? c : p.cols * p.v);
}

// Vectors of v elements: a row of them fits a block or has one pixel; and v divides a sample.
bool rows_fit(uint32_t c, uint32_t v) { return c % v == 0 || c / std::gcd(c, v) <= (uint32_t)kThreads; }
bool usable(uint64_t pixels, uint32_t c, uint32_t v) { return pixels * c % v == 0 && rows_fit(c, v); }
// 16-bit samples of an odd number of elements, which start off a word: shifted vectors of 8 instead of single elements
// cost a few us of prologue and win from 2 to 3 million elements on. Measured forward / backward, bf16, silu: 2 x 100001
// x 37 27 / 45 us against 38 / 70, 4 x 1010615 x 5 56 / 105 against 102 / 181; but 50 x 513 x 65 24 / 30 against 21 / 27,
// and 200 x 501 x 37, above the limit, 37 / 48 against 35 / 47.
// Pairs keep theirs (4 x 300001 x 14 41 / 65 us, shifted 48 / 88), and so does fp32 (2 x 100001 x 37 34 / 51, 33 / 58).
bool shifts(uint64_t n, uint64_t pixels, uint32_t c) {
    return pixels * c % 2 && n * pixels * c >= 5u << 19 && rows_fit(c, 8);
}

uint64_t workspace_floats(uint64_t n, uint64_t pixels, uint32_t c, uint32_t groups, bool bwd) {
    uint64_t most = 0;  // of the cuts that type and alignment may choose
    Plan p;
    for (uint32_t v : {8u, 4u, 2u, 1u})
        for (bool shifted : {false, true})
            if ((shifted ? v == 8 && shifts(n, pixels, c) : usable(pixels, c, v)) &&
                plan_for(n, pixels, c, groups, v, bwd, shifted, p)) {
                const uint64_t w = workspace_of(p, n, c, bwd);
                if (w > most) most = w;
            }
    return most;
}

bsx_status run(bsx_ctx* ctx, Args a, int32_t dtype, const bsx_group_norm_cfg* cfg, void* ws, uint64_t ws_bytes,
               bool bwd, void* stream) {
    if (!ctx || !cfg) return BSX_ERR_INVALID_ARG;
    try {
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
        a.act = cfg->activation;
        a.dropping = cfg->dropout != nullptr;
        if (a.dropping) {
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
        const uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.v | (uintptr_t)a.out;
        uint32_t v = 16 / (uint32_t)size;
        if (all % 16 || !usable(a.pixels, a.c, v)) v = all % (2 * size) == 0 && usable(a.pixels, a.c, 2) ? 2 : 1;
        Plan p;
        bool ok = plan_for(a.n, a.pixels, a.c, a.groups, v, bwd, false, p);
        if (size == 2 && all % 16 == 0 && !p.small && shifts(a.n, a.pixels, a.c))
            ok = plan_for(a.n, a.pixels, a.c, a.groups, v = 8, bwd, true, p);
        if (!ok) return fail(ctx, BSX_ERR_CAPACITY, "too many rows");
        const uint64_t need = workspace_of(p, a.n, a.c, bwd) * 4;
        if (ws_bytes < need || (need && !ws)) return fail(ctx, BSX_ERR_CAPACITY, "the workspace is too small");
        const Call call{&a, &p, (int)(v / std::gcd(a.per, v)), ctx->device, st};
        prof_begin_on(ctx, st);
        const cudaError_t e = dtype == BSX_F32    ? (bwd ? launch_bwd<float>(call) : launch_fwd<float>(call))
                              : dtype == BSX_BF16 ? (bwd ? launch_bwd<__nv_bfloat16>(call) : launch_fwd<__nv_bfloat16>(call))
                                                  : (bwd ? launch_bwd<__half>(call) : launch_fwd<__half>(call));
        if (e != cudaSuccess) {
            cudaGetLastError();
            return check_cuda(ctx, e, bwd ? "launch of norm_bwd_kernel" : "launch of norm_fwd_kernel");
        }
        return post_launch_on(ctx, bwd ? "norm_bwd_kernel" : "norm_fwd_kernel", st);
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
    norm::Args a{};
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
    norm::Args a{};
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
