// Root-mean-square norm of the residual stream, with the residual's addition
// and an e4m3 output with one fp32 scale per token and 128 channels.
//
//   h = x + residual;  residual_out = round(h)
//   y = h / sqrt(mean(h^2) + eps) * weight
//   s = max(max |y| over 128 channels, 1e-30) / 448,  q = e4m3(y / s)
//
// h and every statistic stay in fp32; y is rounded once, to the output type.
// The floor of s keeps 1 / s finite for an all-zero block.  A NaN or infinity
// makes its row's y NaN, hence its scales and codes too.
//
// Bound by bytes (6 flops a value): the row is read once into registers, eight
// values a thread and step, so a block of 128 channels is the eight values of
// half a warp and its maximum four shuffles.
#include <cuda_fp8.h>

#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 1e-30f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Sum over the TPR threads of a row: one warp, or the whole CTA.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (TPR == 32) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    v = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// TPR threads a row (32: a warp each; 0: the CTA), each with CH steps of 8 values.
template <class T, int CH, int TPR>
__global__ void __launch_bounds__(TPR ? 256 : 1024) norm_kernel(sq_norm_args a, bool vec) {
    __shared__ float scratch[32];
    const int tpr = TPR ? TPR : blockDim.x;
    const int64_t row = TPR ? int64_t(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5) : blockIdx.x;
    const int t = TPR ? threadIdx.x & 31 : threadIdx.x;
    if (TPR && row >= a.rows) return;  // whole warps
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    T *res_out = static_cast<T *>(a.residual_out) + row * a.hidden;
    float h[CH][8];
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = (c * tpr + t) * 8, n = min(8, a.hidden - at);
        const bool whole = vec && n == 8;
        if (n > 0) {
            load8(x + at, whole, n, h[c]);
            if (res) {
                float r[8];
                load8(res + at, whole, n, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += r[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = 0.f;
        }
    }
    float factor = 1.f;
    if (a.normalize) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * tpr + t) * 8, n = min(8, a.hidden - at);
            if (res && n > 0) store8(res_out + at, vec && n == 8, n, h[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
        }
        factor = rsqrtf(row_sum<TPR>(squares, scratch) / float(a.hidden) + a.eps);
    }
    const int blocks = (a.hidden + 127) / 128;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = (c * tpr + t) * 8, n = min(8, a.hidden - at);
        const bool whole = vec && n == 8;
        if (a.weight && n > 0) {
            float w[8];
            if (a.weight_dtype == SQ_F32) load8(static_cast<const float *>(a.weight) + at, whole, n, w);
            else if (a.weight_dtype == SQ_BF16) load8(static_cast<const __nv_bfloat16 *>(a.weight) + at, whole, n, w);
            else load8(static_cast<const __half *>(a.weight) + at, whole, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[i];
        }
        if (!a.scale) {
            if (n > 0) store8(static_cast<T *>(a.out) + row * a.hidden + at, whole, n, h[c]);
            continue;
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(h[c][i]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float scale = max_nan(top, kScaleFloor) / kE4m3Max, inverse = 1.f / scale;
        if (n > 0) {
            if ((t & 15) == 0) a.scale[row * blocks + at / 128] = scale;
            uint32_t q[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(h[c][2 * i] * inverse, h[c][2 * i + 1] * inverse),
                                                              __NV_SATFINITE, __NV_E4M3);
                q[i / 2] = i % 2 ? q[i / 2] | two << 16 : two;
            }
            uint8_t *out = static_cast<uint8_t *>(a.out) + row * a.hidden + at;
            if (whole) {
                *reinterpret_cast<uint2 *>(out) = make_uint2(q[0], q[1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < n) out[i] = uint8_t(q[i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

template <class T>
cudaError_t launch_norm(const sq_norm_args &a, cudaStream_t s) {
    const size_t size = sizeof(T);
    auto rows_ok = [&](const void *p, int64_t stride) { return aligned16(p) && stride * size % 16 == 0; };
    const bool vec = a.hidden % 8 == 0 && rows_ok(a.x, a.x_stride) &&
                     (!a.residual || (rows_ok(a.residual, a.residual_stride) && aligned16(a.residual_out))) &&
                     (!a.weight || aligned16(a.weight)) && aligned16(a.out) && a.hidden * size % 16 == 0;
    const int steps = (a.hidden + 7) / 8;
    if (steps <= 64) {  // up to 512 channels: a warp a row, no barrier
        const unsigned grid = unsigned((int64_t(a.rows) + 7) / 8);
        if (steps <= 32) norm_kernel<T, 1, 32><<<grid, 256, 0, s>>>(a, vec);
        else norm_kernel<T, 2, 32><<<grid, 256, 0, s>>>(a, vec);
        return cudaGetLastError();
    }
    // The CTA a row: few rows spread over many threads, many rows two or more steps a thread.
    int ch = a.rows < 592 ? 1 : 2;
    while (ch < 8 && steps > 1024 * ch) ch *= 2;
    const int threads = ((steps + ch - 1) / ch + 31) / 32 * 32;
    const unsigned grid = unsigned(a.rows);
    switch (ch) {
        case 1: norm_kernel<T, 1, 0><<<grid, threads, 0, s>>>(a, vec); break;
        case 2: norm_kernel<T, 2, 0><<<grid, threads, 0, s>>>(a, vec); break;
        case 4: norm_kernel<T, 4, 0><<<grid, threads, 0, s>>>(a, vec); break;
        default: norm_kernel<T, 8, 0><<<grid, threads, 0, s>>>(a, vec); break;
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_rms_norm(const sq_norm_args *args, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_norm_args &a = *args;
    if (a.rows < 0 || a.hidden < 1 || !(a.eps >= 0.f)) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16 || a.weight_dtype < SQ_F32 || a.weight_dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.x_stride < 0 || a.residual_stride < 0) return SQ_ERR_SHAPE;
    if (a.hidden > 65536) return SQ_ERR_UNSUPPORTED;
    if (a.rows == 0) return SQ_OK;
    if (!a.x || !a.out || (a.normalize && !a.weight) || (!a.normalize && (a.weight || a.residual || !a.scale)) ||
        (!a.residual != !a.residual_out))
        return SQ_ERR_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? sq::launch_norm<float>(a, s)
                          : a.dtype == SQ_BF16 ? sq::launch_norm<__nv_bfloat16>(a, s)
                                               : sq::launch_norm<__half>(a, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}
