// Typed access to eight consecutive values, shared by the layer operators
// (norm, convolution, scan, block-scaled product).
#pragma once

#include "sq_common.cuh"

namespace sq {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Eight values starting at p, of which n exist.  width: how many of them one
// access takes, by p's alignment (8: 16-byte accesses, n = 8; 4: four values each,
// n = 4 or 8; 1: singly).  Missing values read as zero.
template <class T>
__device__ __forceinline__ void load8(const T *p, int width, int n, float (&x)[8]) {
    constexpr int kPer = 16 / sizeof(T);
    alignas(16) T v[8];
    if (width == 8 && n == 8) {
#pragma unroll
        for (int i = 0; i < 8; i += kPer) *reinterpret_cast<uint4 *>(v + i) = *reinterpret_cast<const uint4 *>(p + i);
    } else if (width >= 4) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            if (i < n) {
                if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(v + i) = *reinterpret_cast<const uint2 *>(p + i);
                else *reinterpret_cast<uint4 *>(v + i) = *reinterpret_cast<const uint4 *>(p + i);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i + k] = from_float<T>(0.f);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : from_float<T>(0.f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(v[i]);
}

template <class T>
__device__ __forceinline__ void store8(T *p, int width, int n, const float (&x)[8]) {
    constexpr int kPer = 16 / sizeof(T);
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_float<T>(x[i]);
    if (width == 8 && n == 8) {
#pragma unroll
        for (int i = 0; i < 8; i += kPer) *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(v + i);
    } else if (width >= 4) {
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            if (i < n) {
                if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(p + i) = *reinterpret_cast<const uint2 *>(v + i);
                else *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(v + i);
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}

constexpr float kLog2e = 1.4426950408889634f;

// The special function unit's 2^x and 1 / x (two and one units in the last
// place), subnormals flushed to zero.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// x sigmoid(x) = x / (1 + e^-x).  Beyond -88 the exponential is infinite and the
// result -0; -infinity and NaN give NaN as the quotient does.
__device__ __forceinline__ float silu(float x) { return x * reciprocal_approx(1.f + exp2_approx(-kLog2e * x)); }

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace sq
