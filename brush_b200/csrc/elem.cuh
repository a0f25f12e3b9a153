// elem.cuh - element types of the feature operators (dropout.cu, group_norm.cu) and the
// host-side frame of their entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace bsx {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

// One rounding, to nearest even, at the end of 32-bit arithmetic.
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements in the registers they arrive in.
template <class T, int V>
struct Pack {
    static constexpr int kBytes = V * (int)sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes == 32) {
            const uint4 a = __ldg((const uint4*)p), b = __ldg((const uint4*)p + 1);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        } else if constexpr (kBytes == 16) {
            const uint4 a = __ldg((const uint4*)p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else if constexpr (kBytes == 8) {
            const uint2 a = __ldg((const uint2*)p);
            w[0] = a.x, w[1] = a.y;
        } else if constexpr (kBytes == 4) {
            w[0] = __ldg((const uint32_t*)p);
        } else {
            w[0] = __ldg((const uint16_t*)p);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes == 32) {
            ((uint4*)p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            ((uint4*)p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else if constexpr (kBytes == 16) {
            *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
        } else if constexpr (kBytes == 8) {
            *(uint2*)p = make_uint2(w[0], w[1]);
        } else if constexpr (kBytes == 4) {
            *(uint32_t*)p = w[0];
        } else {
            *(uint16_t*)p = (uint16_t)w[0];
        }
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(w[j]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value)
                v[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
            else v[j] = __half2float(__ushort_as_half((unsigned short)(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu)));
        }
    }
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = __float_as_uint(v[j]);
        } else if constexpr (V == 1) {
            const T h = from_f<T>(v[0]);
            w[0] = *reinterpret_cast<const unsigned short*>(&h);
        } else {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[j], v[j + 1]);
                    w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
                    w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        }
    }
};

// Division of numbers up to `most` by one divisor. For most < 2^32 it is a multiplication: with f =
// floor(2^64 / d) + 1 = (2^64 + e) / d, 0 < e <= d, the product's high word is floor(i / d + i e / (d 2^64)),
// and i e / (d 2^64) <= i / 2^64 < 1 / d as long as i d < 2^64.
struct Divisor {
    uint64_t d, f;
    Divisor(uint64_t by, uint64_t most) {
        d = by > most ? most + 1 : by;  // every quotient is 0 either way, and sums of d stay small
        f = most < (1ull << 32) && d > 1 ? UINT64_MAX / d + 1 : 0;
    }
    __device__ __forceinline__ uint64_t of(uint64_t i) const { return f ? __umul64hi(i, f) : i / d; }
};

// The context's device for the duration of one call; the caller's device comes back.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int device) {
        int cur = -1;
        if (cudaGetDevice(&cur) == cudaSuccess && cur != device && cudaSetDevice(device) == cudaSuccess) before = cur;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace bsx
