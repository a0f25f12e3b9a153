// group_norm.cuh - what the group-norm kernels share: arguments, the cut of a tensor into
// blocks, sums over groups inside a block, and the activation.
//
// Layout. A sample is a run of pixels C elements long, read in vectors of V elements. The
// shortest run that starts and ends on a pixel and on a vector has C / gcd(C, V) vectors. A
// "row" is such a run, or for large samples as many of them as a block takes at once, one
// vector a thread: a thread meets the same V channels in every row, so that their weights,
// biases and statistics stay in its registers, odd channel counts included. Rows wider than a
// block, and rows of many channels in small samples, are cut into tiles of columns.
#pragma once

#include "dropout.cuh"
#include "elem.cuh"

namespace bsx {
namespace norm {

constexpr int kThreads = 512;         // most threads of a block
constexpr int kBatch = 8;             // vectors a thread holds, small samples
constexpr int kBatchBwd = 4;          // of x and of v each, backward
// Large samples: rows of a batch, and batches in flight ahead of the one at work; shifted: see Shifted samples below.
__host__ __device__ constexpr int rows_of_batch(bool bwd, bool shifted) { return (bwd ? 2 : 4) / (shifted ? 2 : 1); }
__host__ __device__ constexpr int batches_ahead(bool bwd, bool shifted) { return bwd == shifted ? 2 : 3; }
constexpr uint32_t kMaxBlocks = 512;  // most blocks of a kernel that leaves partial sums

// Division of x by d for x d < 2^32: with f = (2^32 + e) / d, 0 < e <= d, the product's high word is
// floor(x / d + x e / (d 2^32)), and the second term stays below 1 / d. Beyond, a plain division.
struct Div32 {
    uint32_t d, f;
    static Div32 of(uint32_t d, uint64_t most) { return {d, d > 1 && most * d < (1ull << 32) ? (uint32_t)((1ull << 32) / d + 1) : 0}; }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
        return f ? __umulhi(x, f) : d == 1 ? x : x / d;
    }
};

// Kernel arguments: what the first copies need comes first, each 64 bytes of arguments being a miss of its own.
struct Args {
    const void* x;
    const void* v;       // backward: gradient of the output
    uint64_t n, pixels;
    uint32_t c, groups, per;  // per = c / groups
    int param_f32;
    const void* weight;  // null: 1
    const void* bias;    // null: 0
    float* ws;
    void* out;           // forward: out, backward: v_x
    float* mean;
    float* rstd;
    void* v_weight;
    void* v_bias;
    float eps;
    int act, dropping;
    DropArgs drop;
};

// Kernels are compiled for each activation, with and without dropout (ACT, DROP), where their vectors have one or
// two items; the rarer cuts share one that asks at run time (kAny).
constexpr int kAny = 3;
template <int ACT>
__device__ __forceinline__ int act_of(const Args& a) { return ACT == kAny ? a.act : ACT; }
template <int DROP>
__device__ __forceinline__ bool drops(const Args& a) { return DROP == kAny ? a.dropping != 0 : DROP != 0; }

// How the tensor is cut (plan_for in group_norm.cu).
struct Plan {
    uint64_t elems;      // elements of a sample
    uint64_t vecs;       // vectors of a sample
    uint32_t rows;       // rows of a sample
    uint32_t last;       // vectors of its last row
    uint32_t rv;         // vectors of a row
    uint32_t cols;       // vectors of a tile's row; the last tile may have fewer
    uint32_t tiles;
    uint32_t per_unit;   // large samples: blocks of a (tile, sample), which take its rows in turn; or 0:
    uint32_t per_block;  // consecutive rows of a block, over tiles, samples and rows
    uint32_t each, more; // per_unit: rows of a block; of the first `more` blocks, one more
    uint32_t ring;       // batches in shared memory
    uint32_t gl;         // most groups of a tile
    uint32_t k;          // small samples: rows a block takes at a time
    Div32 by_c, by_per, by_cols;
    uint32_t pixels, pixels_last;  // of a row and of a sample's last row
    uint32_t threads, blocks;
    uint32_t v;          // elements of a vector
    uint32_t tail;       // shifted: elements of a sample's last vector where it is not whole, else 0
    int shifted;
    int small;           // one block per (sample, tile), everything in registers
};

template <class T>
__device__ __forceinline__ float param(const void* p, int f32, uint32_t c, float without) {
    if (!p) return without;
    return f32 ? __ldg((const float*)p + c) : to_f(((const T*)p)[c]);
}
// Of V channels from c on, which may run past the last channel (rows of several pixels).
template <class T, int V>
__device__ __forceinline__ void params(const Args& a, const void* p, uint32_t c, float without, float (&to)[V]) {
    if (V > 2 && p && (uintptr_t)p % 16 == 0 && a.c % V == 0) {
        if (a.param_f32) {
            Pack<float, V> raw;
            raw.load((const float*)p + c);
            raw.get(to);
        } else {
            Pack<T, V> raw;
            raw.load((const T*)p + c);
            raw.get(to);
        }
        return;
    }
    uint32_t ch = c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        to[j] = param<T>(p, a.param_f32, ch, without);
        if (++ch == a.c) ch = 0;
    }
}

// Two 32-bit lanes in one instruction, each rounded as the scalar one.
__device__ __forceinline__ void fma2(float& r0, float& r1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;}"
        : "=f"(r0), "=f"(r1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float& r0, float& r1, float a0, float a1, float b0, float b1) {
    asm("{.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;}"
        : "=f"(r0), "=f"(r1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float& r0, float& r1, float a0, float a1, float b0, float b1) {
    asm("{.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;}"
        : "=f"(r0), "=f"(r1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// r = a b + c, a b, a + b over V lanes; an operand of A values has each for V / A lanes.
template <int V, int A, int B, int C>
__device__ __forceinline__ void fma_v(float (&r)[V], const float (&a)[A], const float (&b)[B], const float (&c)[C]) {
    if constexpr (V == 1) r[0] = __fmaf_rn(a[0], b[0], c[0]);
    else
#pragma unroll
        for (int j = 0; j < V; j += 2)
            fma2(r[j], r[j + 1], a[j * A / V], a[(j + 1) * A / V], b[j * B / V], b[(j + 1) * B / V], c[j * C / V], c[(j + 1) * C / V]);
}
template <int V, int A, int B>
__device__ __forceinline__ void mul_v(float (&r)[V], const float (&a)[A], const float (&b)[B]) {
    if constexpr (V == 1) r[0] = __fmul_rn(a[0], b[0]);
    else
#pragma unroll
        for (int j = 0; j < V; j += 2) mul2(r[j], r[j + 1], a[j * A / V], a[(j + 1) * A / V], b[j * B / V], b[(j + 1) * B / V]);
}
template <int V, int A, int B>
__device__ __forceinline__ void add_v(float (&r)[V], const float (&a)[A], const float (&b)[B]) {
    if constexpr (V == 1) r[0] = __fadd_rn(a[0], b[0]);
    else
#pragma unroll
        for (int j = 0; j < V; j += 2) add2(r[j], r[j + 1], a[j * A / V], a[(j + 1) * A / V], b[j * B / V], b[(j + 1) * B / V]);
}
// Sums of V lanes into L items of V / L lanes each, the even and odd lanes of an item apart (kParts sums), so that
// both lanes of a pair add at once.
template <int V, int L>
constexpr int kParts = L == V ? V : 2 * L;
template <int V, int L>
__device__ constexpr int part_of(int j) { return L == V ? j : 2 * (j * L / V) + (j & 1); }
template <int V, int L>
__device__ __forceinline__ void accumulate(float (&sum)[kParts<V, L>], const float (&v)[V]) {
    if constexpr (V == 1) sum[0] += v[0];
    else
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float &s = sum[part_of<V, L>(j)], &s2 = sum[part_of<V, L>(j + 1)];
            add2(s, s2, s, s2, v[j], v[j + 1]);
        }
}
template <int V, int L>
__device__ __forceinline__ void accumulate(float (&sum)[kParts<V, L>], const float (&a)[V], const float (&b)[V]) {
    if constexpr (V == 1) sum[0] = __fmaf_rn(a[0], b[0], sum[0]);
    else
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float &s = sum[part_of<V, L>(j)], &s2 = sum[part_of<V, L>(j + 1)];
            fma2(s, s2, a[j], a[j + 1], b[j], b[j + 1], s, s2);
        }
}
template <int V, int L>
__device__ __forceinline__ void per_item(const float (&part)[kParts<V, L>], float (&item)[L]) {
#pragma unroll
    for (int j = 0; j < L; ++j) item[j] = L == V ? part[j] : part[2 * j] + part[L == V ? 0 : 2 * j + 1];
}

// The approximate exponential and reciprocal (2 and 1 ulp).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// act(z) = z s(w(z)), s the logistic function: w = z (silu), or 2 sqrt(2/pi) (z + 0.044715 z^3)
// (gelu in its tanh form, because (1 + tanh(t)) / 2 = s(2 t)). With e = 2^(-w log2 e) it is
// s = 1 / (1 + e). The special-function unit takes eight cycles for an exponential or reciprocal
// of a warp and would bound a pass over 16-bit data, so two reciprocals are one of the product:
// 1 / a = b / (a b). Exponents are held at 63 so that the product stays finite. What they leave,
// 2^-63, must not be multiplied by a far z, nor by the slope's terms, which grow with it: 2^-62 is
// taken off every s and the result clamped to [0, 1], both in the multiplication that forms it. s is
// off by a few units in the last place, by |w| of them (the rounding of w log2 e) and by 2^-62, and
// is 0 from w = -43 down.
constexpr float kLog2e = 1.4426950408889634f, kGelu1 = 1.5957691216057308f, kGelu3 = 0.044715f;
constexpr float kMostExponent = 63.0f, kLeft = 2.168404344971009e-19f;  // 2^-62
template <int V>
__device__ __forceinline__ void gates(int act, const float (&z)[V], float (&s)[V], float (&e)[V]) {
    constexpr float one[1] = {1.0f};
    if (act == BSX_ACT_SILU) {
        constexpr float k[1] = {-kLog2e};
        mul_v<V>(e, z, k);
    } else {
        constexpr float k1[1] = {-kLog2e * kGelu1}, k3[1] = {-kLog2e * kGelu1 * kGelu3};
        mul_v<V>(e, z, z);
        fma_v<V>(e, e, k3, k1);
        mul_v<V>(e, e, z);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = exp2_fast(fminf(e[j], kMostExponent));
    add_v<V>(s, e, one);
    if constexpr (V == 1) {
        s[0] = __saturatef(rcp_fast(s[0]) - kLeft);
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float r = rcp_fast(s[j] * s[j + 1]), other = s[j];
            s[j] = __saturatef(__fmaf_rn(s[j + 1], r, -kLeft));
            s[j + 1] = __saturatef(__fmaf_rn(other, r, -kLeft));
        }
    }
}
template <int V>
__device__ __forceinline__ void activate(int act, float (&z)[V]) {
    if (act == BSX_ACT_NONE) return;
    float s[V], e[V];
    gates<V>(act, z, s, e);
    mul_v<V>(z, z, s);
}
// v act'(z): act'(z) = s + s (1 - s) z w'(z) = s (1 + c z w'(z)) with c = 1 - s = e s without a difference. NaN goes
// through z. c z is formed first: it is 0 on both sides far from 0, where w' grows without bound but, z being at most
// about kMostBias, stays finite.
template <int V>
__device__ __forceinline__ void back_activate(int act, float (&v)[V], float (&z)[V]) {
    if (act == BSX_ACT_NONE) return;
    constexpr float one[1] = {1.0f};
    float s[V], c[V];
    gates<V>(act, z, s, c);
    mul_v<V>(c, c, s);
    mul_v<V>(c, c, z);
    if (act == BSX_ACT_GELU_TANH) {
        constexpr float k1[1] = {kGelu1}, k3[1] = {3.0f * kGelu1 * kGelu3};
        mul_v<V>(z, z, z);
        fma_v<V>(z, z, k3, k1);
        fma_v<V>(z, z, c, one);
    } else {
        add_v<V>(z, c, one);
    }
    mul_v<V>(z, z, s);
    mul_v<V>(v, v, z);
}
// The slope's z of gelu is formed from biases within this: farther ones (channels switched off by the type's lowest value)
// have the same slope, 0 or 1, and a w' that would overflow. NaN stays.
constexpr float kMostBias = 4611686018427387904.0f;  // 2^62
__device__ __forceinline__ float near_bias(float b) { return b > kMostBias ? kMostBias : b < -kMostBias ? -kMostBias : b; }

// Bit j: element j of a vector at flat element `at` is kept; a vector may lie across two blocks of draws.
template <int V>
__device__ __forceinline__ uint32_t keep_bits(const DropArgs& d, uint32_t step, uint64_t at) {
    uint32_t keep = keep8(d, step, at >> 3) >> (at & 7);
    if ((at & 7) + V > 8) keep |= keep8(d, step, (at >> 3) + 1) << (8 - (at & 7));
    return keep & ((1u << V) - 1u);
}
// drop for V elements from flat element `at`, a multiple of V unless the sample is shifted (S).
template <int V, bool S = false>
__device__ __forceinline__ void drop_vector(const DropArgs& d, uint32_t step, uint64_t at, float (&v)[V]) {
    if constexpr (V == 8 && !S) {
        drop_values<8>(d, step, at >> 3, v);
    } else {
        const uint32_t keep = keep_bits<V>(d, step, at);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = keep >> j & 1u ? v[j] * d.scale : 0.0f;
    }
}

// Zeroes the dropped elements of a packed vector; the kept ones are not scaled.
template <bool S, class T, int V>
__device__ __forceinline__ void drop_packed(const DropArgs& d, uint32_t step, uint64_t at, Pack<T, V>& v) {
    uint32_t keep;
    if constexpr (V == 8 && !S) {
        const uint32_t q0 = (uint32_t)(at >> 3), q1 = (uint32_t)(at >> 35);
        const uint4 w = philox7(d, q0, q1, step, 0u);
        if (!any_tie(d, w)) {
            const uint32_t top = d.t_hi << 16 | 0xffffu, word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v.w[k] &= (word[k] << 16 > top ? 0xffffu : 0u) | (word[k] > top ? 0xffff0000u : 0u);
            return;
        }
        keep = tie_bits(d, step, q0, q1, w);
    } else {
        keep = keep_bits<V>(d, step, at);
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (!(keep >> j & 1u)) {
            if constexpr (sizeof(T) == 4) v.w[j] = 0u;
            else v.w[j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
}

// The columns and groups of a tile. A vector has L items of V / L elements, each in one group.
struct Tile {
    uint32_t cols;         // vectors in the tile's row
    uint32_t c0, c1;       // channels
    uint32_t g0, groups;   // groups that have channels here
    uint32_t stride;       // items from a channel to its next copy in the block
    uint32_t copies;       // copies of the channels in the block's k rows
    uint32_t lanes, log;   // threads that add up a group: 2^log
};
template <int V, int L>
__device__ __forceinline__ Tile tile_of(const Args& a, const Plan& p, uint32_t t) {
    Tile r;
    if (p.tiles == 1) {
        r.cols = p.cols;
        r.c0 = 0, r.c1 = a.c;
        r.g0 = 0, r.groups = a.groups;
        r.stride = a.c / (V / L);
        r.copies = p.by_c(p.k * p.cols * V);
    } else {
        r.cols = min(p.cols, p.rv - t * p.cols);
        r.c0 = t * p.cols * V, r.c1 = r.c0 + r.cols * V;
        r.g0 = p.by_per(r.c0);
        r.groups = p.by_per(r.c1 - 1) - r.g0 + 1;
        r.stride = r.cols * L;
        r.copies = p.k;
    }
    const uint32_t each = blockDim.x / r.groups;
    r.log = each ? 31 - __clz(each) : 0;
    r.lanes = 1u << r.log;
    return r;
}
// Channels of group g0 + q in the tile, in items from c0: [lo, hi).
template <int V, int L>
__device__ __forceinline__ void group_span(const Args& a, const Tile& t, uint32_t q, uint32_t& lo, uint32_t& hi) {
    const uint32_t first = (t.g0 + q) * a.per;
    lo = (max(first, t.c0) - t.c0) / (V / L);
    hi = (min(first + a.per, t.c1) - t.c0) / (V / L);
}

// Place of an item in shared memory: with several items a thread, four words more every 32, so that threads write
// 16 bytes at a time and the walks over copies of a group's items meet other banks.
template <int L>
__device__ __forceinline__ uint32_t place(uint32_t e) { return L > 1 ? e + (e >> 5) * 4 : e; }
template <int L>
__host__ __device__ constexpr uint32_t places(uint32_t threads) { return L > 1 ? threads * L + threads * L / 8 : threads; }
template <int L>
__device__ __forceinline__ void put_items(float* part, const float (&x)[L], bool active) {
    if constexpr (L >= 4) {
        float4* to = (float4*)(part + place<L>(threadIdx.x * L));  // L items lie in one run of 32
#pragma unroll
        for (int j = 0; j < L; j += 4)
            to[j / 4] = active ? make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    } else {
#pragma unroll
        for (int j = 0; j < L; ++j) part[place<L>(threadIdx.x * L + j)] = active ? x[j] : 0.0f;
    }
}

// A thread's part in the sums over the tile's groups: the items of group `q` that it walks.
struct GroupWalk {
    uint32_t q, l;        // group, and place among the group's t.lanes threads
    uint32_t at, m, i;    // first item, its copy and place in the group
    uint32_t dm, di, width;
};
template <int V, int L>
__device__ __forceinline__ GroupWalk group_walk(const Args& a, const Tile& t, uint32_t u) {
    GroupWalk w;
    w.q = u >> t.log, w.l = u & (t.lanes - 1);
    uint32_t lo, hi;
    group_span<V, L>(a, t, min(w.q, t.groups - 1), lo, hi);
    w.width = hi - lo;
    const float inv = 1.0f / (float)w.width;  // quotients below 2^10, half a unit from the next: exact
    w.m = (uint32_t)(((float)w.l + 0.5f) * inv);
    w.i = w.l - w.m * w.width;
    w.at = w.m * t.stride + lo + w.i;
    w.dm = (uint32_t)(((float)t.lanes + 0.5f) * inv);
    w.di = t.lanes - w.dm * w.width;
    return w;
}

// Sums over the tile's groups of one value per item (thread t holds items t L ... t L + L - 1 of the block's
// rows), in a fixed order: t.lanes threads walk each group's items (`mine`: group_walk of the thread). Afterwards
// sum[q] holds group g0 + q for all threads. Starts without a barrier (whoever read part or sum last has passed one
// since, or passes the first one here before they are written); ends with one.
template <int V, int L, bool PAIR>
__device__ __forceinline__ void group_sums(const Args& a, const Tile& t, const GroupWalk& mine, const float (&x)[L],
                                           const float (&y)[L], bool active, float* part, float2* warp_sum, float2* sum) {
    const uint32_t tid = threadIdx.x, half = places<L>(blockDim.x);  // half: the pair's second values
    put_items<L>(part, x, active);
    if (PAIR) put_items<L>(part + half, y, active);
    __syncthreads();
    const uint32_t in = min(t.lanes, 32u);
    for (uint32_t base = 0; base < t.groups * t.lanes; base += blockDim.x) {
        GroupWalk w = mine;
        if (base) w = group_walk<V, L>(a, t, base + tid);
        float s = 0.0f, s2 = 0.0f;
        if (w.q < t.groups)
            while (w.m < t.copies) {
                s += part[place<L>(w.at)];
                if (PAIR) s2 += part[half + place<L>(w.at)];
                w.m += w.dm, w.i += w.di;
                w.at += w.dm * t.stride + w.di;
                if (w.i >= w.width) w.i -= w.width, ++w.m, w.at += t.stride - w.width;
            }
        for (uint32_t o = in / 2; o; o /= 2) {
            s += __shfl_xor_sync(~0u, s, o);
            if (PAIR) s2 += __shfl_xor_sync(~0u, s2, o);
        }
        if (t.lanes <= 32) {
            if (w.l == 0 && w.q < t.groups) sum[w.q] = make_float2(s, s2);
        } else if ((tid & 31) == 0) {
            warp_sum[tid / 32] = make_float2(s, s2);
        }
    }
    __syncthreads();
    if (t.lanes > 32) {
        if (tid < t.groups) {
            float s = 0.0f, s2 = 0.0f;
            for (uint32_t w = 0; w < t.lanes / 32; ++w) {
                const float2 v = warp_sum[tid * (t.lanes / 32) + w];
                s += v.x;
                s2 += v.y;
            }
            sum[tid] = make_float2(s, s2);
        }
        __syncthreads();
    }
}

// First channel of item j of a vector that starts at channel c.
template <int V, int L>
__device__ __forceinline__ uint32_t channel_at(const Args& a, uint32_t c, int j) {
    uint32_t ch = c + j * (V / L);
    if (j > 0) while (ch >= a.c) ch -= a.c;  // rows of several pixels
    return ch;
}

// Large samples. Rows are whole block iterations, numbered over tiles, samples ("units") and rows. A block has
// parts of the units first ... last ("segments"): every per_unit-th row of one unit (grid per_unit x units), or
// consecutive rows (grid blocks x 1).
struct Run {
    uint32_t first, last;
    uint32_t w0, w1;  // first row of the unit, or consecutive rows
    uint32_t stride;  // rows from one to the next
};
__device__ __forceinline__ uint32_t block_id() { return blockIdx.y * gridDim.x + blockIdx.x; }
__device__ __forceinline__ Run run_of(const Args& a, const Plan& p) {
    if (p.per_unit) return {blockIdx.y, blockIdx.y, blockIdx.x, 0, p.per_unit};
    const uint32_t total = p.rows * (uint32_t)a.n * p.tiles, w0 = blockIdx.x * p.per_block, w1 = min(w0 + p.per_block, total);
    return {w0 / p.rows, (w1 - 1) / p.rows, w0, w1, 1};
}
// Rows r0, r0 + stride, ... of unit u in a run; ends: the unit's last row among them.
struct Rows {
    uint32_t r0, iters;
    bool ends;
};
__device__ __forceinline__ Rows rows_of(const Plan& p, const Run& run, uint32_t u) {
    if (p.per_unit) {
        const bool extra = run.w0 < p.more;
        return {run.w0, p.each + extra, p.more ? run.w0 + 1 == p.more : run.w0 + 1 == p.per_unit};
    }
    const uint32_t from = max(u * p.rows, run.w0), to = min((u + 1) * p.rows, run.w1);
    return {from - u * p.rows, to - from, to == (u + 1) * p.rows};
}
// Pixels of a block's part of a unit (of a tile of one pixel a row: rows).
__device__ __forceinline__ float pixels_of(const Plan& p, const Rows& r) {
    return (float)(r.iters - r.ends) * (float)p.pixels + (r.ends ? (float)p.pixels_last : 0.0f);
}
// Blocks that have rows of unit u: [b0, b1].
__device__ __forceinline__ void runs_of_unit(const Plan& p, uint32_t u, uint32_t& b0, uint32_t& b1) {
    if (p.per_unit) {
        b0 = u * p.per_unit;
        b1 = b0 + p.per_unit - 1;
    } else {
        b0 = u * p.rows / p.per_block;
        b1 = ((u + 1) * p.rows - 1) / p.per_block;
    }
}
struct Segment {
    uint32_t n, tile, c;      // sample, tile, channel of the thread's first element
    Rows rows;
    uint32_t iters, cnt;      // rows; of this thread, which misses at most a sample's last row
    uint32_t tail;            // shifted: the row, from 1, whose vector of this thread has p.tail elements; 0: none
    uint64_t at;              // first element of the thread's vector in the first row
};
template <int V>
__device__ __forceinline__ Segment segment_of(const Args& a, const Plan& p, const Run& run, uint32_t u, const Tile& t) {
    Segment s;
    s.tile = p.tiles == 1 ? 0 : u / (uint32_t)a.n;
    s.n = u - s.tile * (uint32_t)a.n;
    s.rows = rows_of(p, run, u);
    s.iters = s.rows.iters;
    const uint32_t col = s.tile * p.cols + threadIdx.x;
    s.cnt = threadIdx.x < t.cols ? s.iters - (s.rows.ends && col >= p.last) : 0;
    s.at = s.n * p.elems + ((uint64_t)s.rows.r0 * p.rv + col) * V;
    s.tail = p.tail && s.rows.ends && col + 1 == p.last ? s.iters : 0;
    s.c = col * V;
    if (p.tiles == 1) s.c -= p.by_c(s.c) * a.c;
    return s;
}
// Batches of R rows of a run, each inside one segment.
template <int R>
__device__ __forceinline__ uint32_t batches_of(const Plan& p, const Run& run) {
    uint32_t all = 0;
    for (uint32_t u = run.first; u <= run.last; ++u) {
        all += (rows_of(p, run, u).iters + R - 1) / R;
    }
    return all;
}
// The batch that is copied next: a walk over a run's batches, forwards or backwards.
template <int V, int R>
struct Walk {
    uint32_t u, i, iters, valid;  // unit; first row of the batch, of the segment's iters; rows in which the thread has a vector
    uint64_t at;                  // element of row i

    __device__ __forceinline__ void unit(const Args& a, const Plan& p, const Run& run, bool last) {
        const Rows r = rows_of(p, run, u);
        iters = r.iters;
        i = last ? (iters - 1) / R * R : 0;
        const uint32_t tile = p.tiles == 1 ? 0 : u / (uint32_t)a.n, n = u - tile * (uint32_t)a.n;
        const uint32_t col = tile * p.cols + threadIdx.x;
        valid = threadIdx.x < p.cols && col < p.rv ? iters - (r.ends && col >= p.last) : 0;
        at = n * p.elems + ((uint64_t)(r.r0 + i * run.stride) * p.rv + col) * V;
    }
    __device__ __forceinline__ void next(const Args& a, const Plan& p, const Run& run, uint64_t step) {
        i += R;
        at += R * step;
        if (i >= iters && u < run.last) {
            ++u;
            unit(a, p, run, false);
        }
    }
    __device__ __forceinline__ void before(const Args& a, const Plan& p, const Run& run, uint64_t step) {
        if (i) {
            i -= R;
            at -= R * step;
        } else if (u > run.first) {
            --u;
            unit(a, p, run, true);
        }
    }
    // Back to batch `to` of a run of `all`.
    __device__ __forceinline__ void rewind(const Args& a, const Plan& p, const Run& run, uint64_t step, uint32_t all, uint32_t to) {
        u = run.last;
        unit(a, p, run, true);
        if (run.first == run.last) {
            at -= (uint64_t)(i - to * R) * step;
            i = to * R;
        } else {
            for (uint32_t b = all - 1; b > to; --b) before(a, p, run, step);
        }
    }
};

// Copies into a thread's own places of shared memory, which it alone reads: no barrier, only its own wait. A copy
// takes at least 4 bytes: of a single 16-bit element the aligned word that holds it is copied, and `read` picks its
// half. The word's other half is read only if it belongs to the tensor too: words start inside it where the tensor
// starts on 4 bytes (otherwise the element is loaded and stored), and a last half word is copied alone.
template <class T, int V>
__device__ __forceinline__ void copy_async(Pack<T, V>* to, const T* base, uint64_t at, uint64_t count) {
    constexpr int bytes = V * (int)sizeof(T);
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (bytes == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(base + at) : "memory");
    } else if constexpr (bytes >= 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(base + at), "n"(bytes) : "memory");
    } else if ((uintptr_t)base % 4 == 0) {
        const uint64_t word = at & ~(uint64_t)1;
        const uint32_t have = word + 1 < count ? 4u : 2u;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(base + word), "r"(have) : "memory");
    } else {
        Pack<T, V> v;
        v.load(base + at);
        v.w[0] |= v.w[0] << 16;  // in both halves
        *to = v;
    }
}
template <class T, int V>
__device__ __forceinline__ Pack<T, V> read(const Pack<T, V>* from, uint64_t at) {
    Pack<T, V> v = *from;
    if constexpr (V * sizeof(T) == 2)
        if (at & 1) v.w[0] >>= 16;
    return v;
}

// Shifted samples (16-bit types, an odd number of elements): samples after the first start off a vector, or a word.
// Their vectors are still counted from the sample's own start, so that channels, rows and pixels fall as they do
// elsewhere, but lie across two aligned ones: a thread copies both, takes its elements out of the two, and passes
// what reaches into the next aligned vector to its neighbour when it stores. The last vector may have fewer elements.
// What that buys was measured where it is chosen (shifts in group_norm.cu).

// V elements of two neighbouring aligned vectors from element `off` (< V) on.
template <class T, int V>
__device__ __forceinline__ Pack<T, V> across(const Pack<T, V>& lo, const Pack<T, V>& hi, uint32_t off) {
    const uint32_t bytes = off * (uint32_t)sizeof(T), odd = bytes & 2u;
    Pack<T, V> r;
    const auto take = [&](const uint32_t(&w)[5]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.w[k] = odd ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
    };
    switch (bytes >> 2) {  // the same for a whole row
        case 0: take({lo.w[0], lo.w[1], lo.w[2], lo.w[3], hi.w[0]}); break;
        case 1: take({lo.w[1], lo.w[2], lo.w[3], hi.w[0], hi.w[1]}); break;
        case 2: take({lo.w[2], lo.w[3], hi.w[0], hi.w[1], hi.w[2]}); break;
        default: take({lo.w[3], hi.w[0], hi.w[1], hi.w[2], hi.w[3]}); break;
    }
    return r;
}
// Copy of the vector at element `at` of a tensor of `count`, and the vector itself once it has arrived.
template <class T, int V, bool S>
__device__ __forceinline__ void copy_vector(Pack<T, V>* to, const T* base, uint64_t at, uint64_t count) {
    if constexpr (!S) {
        copy_async<T, V>(to, base, at, count);
    } else {
        const uint64_t first = at & ~(uint64_t)(V - 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint64_t e = first + k * V;
            const uint32_t have = e >= count ? 0u : count - e < V ? (uint32_t)(count - e) * (uint32_t)sizeof(T) : 16u;
            if (have)  // what lies behind the tensor is not read
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + k * blockDim.x)),
                             "l"(base + e), "r"(have) : "memory");
        }
    }
}
template <class T, int V, bool S>
__device__ __forceinline__ Pack<T, V> read_vector(const Pack<T, V>* from, uint64_t at) {
    if constexpr (S) return across<T, V>(from[0], from[blockDim.x], (uint32_t)at & (V - 1));
    else return read<T, V>(from, at);
}
// Elements from `valid` on become 0.
template <int V>
__device__ __forceinline__ void cut(float (&f)[V], uint32_t valid) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = j < valid ? f[j] : 0.0f;
}
template <class T, int V>
__device__ __forceinline__ void store_elements(T* out, uint64_t at, const Pack<T, V>& o, uint32_t from, uint32_t to) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j >= from && j < to) {
            ((uint16_t*)out)[at + j] = (uint16_t)(j & 1 ? o.w[j / 2] >> 16 : o.w[j / 2]);
        }
}
// Stores the first `valid` elements of a vector for every thread of a warp with ok; neighbouring threads have
// neighbouring vectors. All threads of the warp call it.
template <class T, int V>
__device__ __forceinline__ void store_shifted(T* out, uint64_t at, const Pack<T, V>& o, bool ok, uint32_t valid) {
    const uint32_t lane = threadIdx.x & 31, shift = (uint32_t)at & (V - 1), own = V - shift;  // own: of the vector it starts in
    Pack<T, V> before;
#pragma unroll
    for (int k = 0; k < 4; ++k) before.w[k] = __shfl_up_sync(~0u, o.w[k], 1);
    const uint32_t oks = __ballot_sync(~0u, ok);
    if (!ok) return;
    const bool left = lane > 0 && (oks >> (lane - 1) & 1u), right = lane < 31 && (oks >> (lane + 1) & 1u);
    if (shift == 0) {
        if (valid == V) o.store(out + at);
        else store_elements(out, at, o, 0, valid);
        return;
    }
    if (left && valid >= own) {
        across<T, V>(before, o, own).store(out + (at - shift));
    } else {
        if (left) store_elements(out, at - V, before, own, V);
        store_elements(out, at, o, 0, valid < own ? valid : own);
    }
    if (!right) store_elements(out, at, o, own, valid);  // nobody to pass them to
}

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// Joins what the blocks of a unit left for its tile's groups: thread (l, q) takes group q of every each-th block,
// f(pair, count of values, q, s, s2) adds to its two sums, and sum[q] holds the totals for all threads.
template <int V, class F>
__device__ __forceinline__ void join_runs(const Args& a, const Plan& p, const Tile& t, uint32_t n, const float2* slots,
                                          float* part, float2* sum, F f) {
    const uint32_t tid = threadIdx.x, threads = blockDim.x, tile_c = p.tiles == 1 ? a.c : p.cols * V;
    for (uint32_t q0 = 0; q0 < t.groups; q0 += threads) {
        const uint32_t groups = min(t.groups - q0, threads), each = threads / groups;
        const uint32_t l = tid / groups, q = q0 + tid - l * groups;
        float s = 0.0f, s2 = 0.0f;
        if (l < each && p.per_unit && p.tiles == 1) {  // every per_unit-th row: counts differ by one row
            const float px = (float)p.pixels * (float)a.per, less = (float)p.each * px;
            const uint32_t ends = p.more ? p.more - 1 : p.per_unit - 1;  // the block with the unit's last row
            const float cut = (float)(p.pixels - p.pixels_last) * (float)a.per;
            const float2* from = slots + (uint64_t)(n * p.per_unit + n + l) * p.gl + q;
            constexpr int G = 4;  // loads in flight
            for (uint32_t j = l; j < p.per_unit; j += G * each, from += (uint64_t)(G * each) * p.gl) {
                float2 v[G];
#pragma unroll
                for (int i = 0; i < G; ++i)
                    if (j + i * each < p.per_unit) v[i] = __ldcg(from + (uint64_t)(i * each) * p.gl);
#pragma unroll
                for (int i = 0; i < G; ++i)
                    if (j + i * each < p.per_unit) {
                        const float count = (j + i * each < p.more ? less + px : less) - (j + i * each == ends ? cut : 0.0f);
                        f(v[i], count, q, s, s2);
                    }
            }
        } else if (l < each) {
            const uint32_t grp = t.g0 + q;
            const uint32_t t0 = p.tiles == 1 ? 0 : grp * a.per / tile_c;
            const uint32_t t1 = p.tiles == 1 ? 0 : ((grp + 1) * a.per - 1) / tile_c;
#pragma unroll 1
            for (uint32_t k = t0; k <= t1; ++k) {
                const uint32_t u = k * (uint32_t)a.n + n, at = grp - (p.tiles == 1 ? 0 : p.by_per(k * tile_c));
                const uint32_t width = p.tiles == 1 ? a.per
                                                    : min((grp + 1) * a.per, min((k + 1) * tile_c, a.c)) - max(grp * a.per, k * tile_c);
                uint32_t b0, b1;
                runs_of_unit(p, u, b0, b1);
#pragma unroll 1
                for (uint32_t b = b0 + l; b <= b1; b += each) {
                    const float2 v = __ldcg(slots + (uint64_t)(b + u) * p.gl + at);
                    const Run run = p.per_unit ? Run{u, u, b - b0, 0, 1} : Run{u, u, b * p.per_block, b * p.per_block + p.per_block, 1};
                    f(v, pixels_of(p, rows_of(p, run, u)) * (float)width, q, s, s2);
                }
            }
        }
        part[tid] = s;
        part[threads + tid] = s2;
        __syncthreads();
        uint32_t rows = each;  // of `groups` values: halved until few are left
        while (rows > 4) {
            const uint32_t half = (rows + 1) / 2;
            if (l + half < rows) {
                part[tid] += part[tid + half * groups];
                part[threads + tid] += part[threads + tid + half * groups];
            }
            rows = half;
            __syncthreads();
        }
        if (tid < groups) {
            float r = 0.0f, r2 = 0.0f;
            for (uint32_t m = 0; m < rows; ++m) {
                r += part[m * groups + tid];
                r2 += part[threads + m * groups + tid];
            }
            sum[q0 + tid] = make_float2(r, r2);
        }
        __syncthreads();
    }
}

// Host side, one per element type and direction (group_norm_{fwd,bwd}_{f32,bf16,f16}.cu). items: L above.
struct Call {
    const Args* a;
    Plan* p;
    int items;
    int device;
    cudaStream_t stream;
};
template <class T>
cudaError_t launch_fwd(const Call& c);
template <class T>
cudaError_t launch_bwd(const Call& c);

}  // namespace norm
}  // namespace bsx
