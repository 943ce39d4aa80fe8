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
// half a warp and its maximum four shuffles.  Measured, bf16 with residual and
// e4m3 output: 65536 x 5120 in 397 us (5.9 TB/s, 0.92 of the measured copy; with a
// CTA a row and nothing on its way 560 us), one row of 5120 in 2.7 us, of launch
// and two trips to memory; 777 x 4100 f16 (rows on 8-byte boundaries) 6.0 us.
#include <cuda_fp8.h>

#include "sq_vec.cuh"

namespace sq {
int sms_of(cudaStream_t stream);  // sq_fast.cu
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

// Eight weights from `at` on.
__device__ __forceinline__ void load_weights(const sq_norm_args &a, int at, int width, int n, float (&w)[8]) {
    if (a.weight_dtype == SQ_F32) load8(static_cast<const float *>(a.weight) + at, width, n, w);
    else if (a.weight_dtype == SQ_BF16) load8(static_cast<const __nv_bfloat16 *>(a.weight) + at, width, n, w);
    else load8(static_cast<const __half *>(a.weight) + at, width, n, w);
}

// Eight outputs of a row: in T, or e4m3 with the scale of their 128 channels
// (the eight values of 16 neighbouring lanes; every lane of the warp calls).
template <class T>
__device__ __forceinline__ void put(const sq_norm_args &a, int64_t row, int at, int width, int n, const float (&y)[8]) {
    if (!a.scale) {
        if (n > 0) store8(static_cast<T *>(a.out) + row * a.hidden + at, width, n, y);
        return;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(y[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = max_nan(top, kScaleFloor) / kE4m3Max, inverse = 1.f / scale;
    if (n <= 0) return;
    if ((threadIdx.x & 15) == 0) a.scale[row * ((a.hidden + 127) / 128) + at / 128] = scale;
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inverse, y[2 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
        q[i / 2] = i % 2 ? q[i / 2] | two << 16 : two;
    }
    uint8_t *out = static_cast<uint8_t *>(a.out) + row * a.hidden + at;
    if (width == 8 && n == 8) {
        *reinterpret_cast<uint2 *>(out) = make_uint2(q[0], q[1]);
    } else if (width >= 4) {
        reinterpret_cast<uint32_t *>(out)[0] = q[0];
        if (n > 4) reinterpret_cast<uint32_t *>(out)[1] = q[1];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) out[i] = uint8_t(q[i / 4] >> (8 * (i % 4)));
    }
}

// TPR threads a row (32: a warp each; 0: the CTA), each with CH steps of 8 values.
template <class T, int CH, int TPR>
__global__ void __launch_bounds__(TPR ? 256 : 1024) norm_kernel(sq_norm_args a, int width) {
    __shared__ float scratch[32];
    const int tpr = TPR ? TPR : blockDim.x;
    const int64_t row = TPR ? int64_t(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5) : blockIdx.x;
    const int t = TPR ? threadIdx.x & 31 : threadIdx.x;
    if (TPR && row >= a.rows) return;  // whole warps
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    float h[CH][8];
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = (c * tpr + t) * 8, n = min(8, a.hidden - at);
        if (n > 0) {
            load8(x + at, width, n, h[c]);
            if (res) {
                float r[8];
                load8(res + at, width, n, r);
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
            if (res && n > 0) store8(static_cast<T *>(a.residual_out) + row * a.hidden + at, width, n, h[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
        }
        factor = rsqrtf(row_sum<TPR>(squares, scratch) / float(a.hidden) + a.eps);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = (c * tpr + t) * 8, n = min(8, a.hidden - at);
        if (a.weight && n > 0) {
            float w[8];
            load_weights(a, at, width, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[i];
        }
        put<T>(a, row, at, width, n, h[c]);
    }
}

// Many rows of 16-byte aligned pieces: persistent CTAs, kRows rows on their way.
// Each thread copies (cp.async) what it will itself read, so the only barrier of
// a row is its sum's; the weights stay in registers.
constexpr int kRows = 3;

template <class T, int CH>
__global__ void __launch_bounds__(512) norm_rows_kernel(sq_norm_args a) {
    extern __shared__ __align__(16) unsigned char ring[];  // [kRows][x, residual][CH][threads][8 values]
    __shared__ float scratch[2][32];
    const int t = threadIdx.x, threads = blockDim.x;
    constexpr int kPiece = 8 * sizeof(T);
    float w[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = (c * threads + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[c][i] = 0.f;
        if (at < a.hidden) load_weights(a, at, 8, 8, w[c]);
    }
    auto slot = [&](int stage, int which, int c) { return ring + int64_t((((stage * 2 + which) * CH + c) * threads + t)) * kPiece; };
    auto fetch = [&](int64_t row, int stage) {
        if (row < a.rows) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                const T *from = which ? static_cast<const T *>(a.residual) : static_cast<const T *>(a.x);
                if (!from) continue;
                from += row * (which ? a.residual_stride : a.x_stride);
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int at = (c * threads + t) * 8;
                    if (at >= a.hidden) continue;
#pragma unroll
                    for (int i = 0; i < kPiece; i += 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n"
                                     ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(slot(stage, which, c) + i))),
                                     "l"(reinterpret_cast<const unsigned char *>(from + at) + i) : "memory");
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i + 1 < kRows; ++i) fetch(blockIdx.x + int64_t(i) * gridDim.x, i);
    int stage = 0, turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        fetch(row + int64_t(kRows - 1) * gridDim.x, (stage + kRows - 1) % kRows);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(kRows - 1) : "memory");
        float h[CH][8], squares = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * threads + t) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = 0.f;
            if (at >= a.hidden) continue;
            load8(reinterpret_cast<const T *>(slot(stage, 0, c)), 8, 8, h[c]);
            if (a.residual) {
                float r[8];
                load8(reinterpret_cast<const T *>(slot(stage, 1, c)), 8, 8, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += r[i];
                store8(static_cast<T *>(a.residual_out) + row * a.hidden + at, 8, 8, h[c]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
        }
        const float factor = rsqrtf(row_sum<0>(squares, scratch[turn]) / float(a.hidden) + a.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * threads + t) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[c][i];
            put<T>(a, row, at, 8, min(8, a.hidden - at), h[c]);
        }
        stage = stage + 1 == kRows ? 0 : stage + 1;
        turn ^= 1;
    }
}

template <class T, int CH>
cudaError_t launch_rows(const sq_norm_args &a, int threads, int bytes, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(norm_rows_kernel<T, CH>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    int each = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, norm_rows_kernel<T, CH>, threads, bytes);
    if (e != cudaSuccess) return e;
    const int64_t grid = int64_t(sms_of(s)) * each;
    norm_rows_kernel<T, CH><<<unsigned(grid < 1 ? 1 : grid < a.rows ? grid : a.rows), threads, bytes, s>>>(a);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_norm(const sq_norm_args &a, cudaStream_t s) {
    const int64_t size = sizeof(T);
    auto fits = [&](int n) {  // rows of pieces of n values, each by one access
        auto on = [&](const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (bytes < 16 ? bytes : 16) == 0; };
        return a.hidden % n == 0 && a.x_stride % n == 0 && on(a.x, n * size) &&
               (!a.residual || (a.residual_stride % n == 0 && on(a.residual, n * size) && on(a.residual_out, n * size))) &&
               on(a.weight, n * (a.weight_dtype == SQ_F32 ? 4 : 2)) && on(a.out, n * (a.scale ? 1 : size));
    };
    const int width = fits(8) ? 8 : fits(4) ? 4 : 1;
    const int steps = (a.hidden + 7) / 8;
    if (steps <= 64) {  // up to 512 channels: a warp a row, no barrier
        const unsigned grid = unsigned((int64_t(a.rows) + 7) / 8);
        if (steps <= 32) norm_kernel<T, 1, 32><<<grid, 256, 0, s>>>(a, width);
        else norm_kernel<T, 2, 32><<<grid, 256, 0, s>>>(a, width);
        return cudaGetLastError();
    }
    // Rows on their way while others are worked on, once each resident CTA has several.
    if (width == 8 && a.normalize && a.rows >= 2048 && steps <= 2048) {
        const int ch = steps <= 1024 ? 2 : 4, threads = ((steps + ch - 1) / ch + 31) / 32 * 32;
        const int bytes = kRows * 2 * ch * threads * 8 * int(size);
        if (bytes <= 200 * 1024)
            return ch == 2 ? launch_rows<T, 2>(a, threads, bytes, s) : launch_rows<T, 4>(a, threads, bytes, s);
    }
    // The CTA a row: few rows spread over many threads, many rows two or more steps a thread.
    int ch = a.rows < 592 ? 1 : 2;
    while (ch < 8 && steps > 1024 * ch) ch *= 2;
    const int threads = ((steps + ch - 1) / ch + 31) / 32 * 32;
    const unsigned grid = unsigned(a.rows);
    switch (ch) {
        case 1: norm_kernel<T, 1, 0><<<grid, threads, 0, s>>>(a, width); break;
        case 2: norm_kernel<T, 2, 0><<<grid, threads, 0, s>>>(a, width); break;
        case 4: norm_kernel<T, 4, 0><<<grid, threads, 0, s>>>(a, width); break;
        default: norm_kernel<T, 8, 0><<<grid, threads, 0, s>>>(a, width); break;
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
