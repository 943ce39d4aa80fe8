// Conversions and approximate functions shared by the layer operators (norm,
// convolution, scan, block-scaled product).
#pragma once

#include "sq_common.cuh"

namespace sq {

// SMs that kernels launched on `stream` can run on (sq_fast.cu); 0 when the device cannot be asked.
int sms_of(cudaStream_t stream);

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

// x sigmoid(x) = x / (1 + e^-x).  Below -87.3 the reciprocal is flushed to zero and the
// result is -0, for less than 10^-36 in size; -infinity and NaN give NaN as the quotient does.
__device__ __forceinline__ float silu(float x) { return x * reciprocal_approx(1.f + exp2_approx(-kLog2e * x)); }

// Pairs of fp32 values, one instruction for both.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return reinterpret_cast<float2 &>(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r) : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return reinterpret_cast<float2 &>(r);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace sq
