// Root-mean-square norm of the residual stream, with the residual's addition
// and an e4m3 output with one fp32 scale per token and 128 channels.
//
//   h = x + residual;  residual_out = round(h)
//   y = h / sqrt(mean(h^2) + eps) * weight
//   s = max(max |y| over 128 channels, 1e-30) / 448,  q = e4m3(y / s)
//
// h and every statistic stay in fp32; y is rounded once, to the output type.
// The floor of s keeps 1 / s finite for an all-zero block.  Rows whose squares
// overflow (|h| above 1.8e19) take them of h times 2^-80.  A NaN makes its row's y
// NaN, an infinity its own channel's, with the scale and codes of their blocks; the
// other channels of an infinite row are 0.
//
// Bound by bytes (6 flops a value): the row is read once into registers, eight
// values a thread and step, so a block of 128 channels is the eight values of
// half a warp and its maximum four shuffles.  Measured, bf16 with residual and
// e4m3 output: 65536 x 5120 in 385 us (6.1 TB/s, 0.95 of the measured copy; with a
// CTA a row and nothing on its way 560 us), one row of 5120 in 2.8 us, of launch
// and two trips to memory; 777 x 4100 f16 (rows on 8-byte boundaries) 6.1 us;
// quantization alone, a CTA a row, of 65536 x 4096 156 us (5.1 TB/s).
#include <cuda_fp8.h>

#include <type_traits>

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

// x / 448, correctly rounded for normal x of 1e-30 and above: the product with the rounded
// 1 / 448 is a faithful quotient, and its remainder makes it the rounded one (Markstein, IBM J.
// Res. Dev. 34, 1990).
__device__ __forceinline__ float over_most(float x) {
    constexpr float inverse = 1.f / kE4m3Max;
    const float q = x * inverse;
    return x == INFINITY ? x : fmaf(fmaf(-kE4m3Max, q, x), inverse, q);
}

// y / s of two values in the same way, from an approximate 1 / s: off by less than 0.5001 units
// in the last place.  (The product alone is off by up to 2, which moves a code where y / s lies at
// a tie of two codes; a division a value took 507 us for 388 at 65536 x 5120.)
__device__ __forceinline__ float2 quotients(float2 y, float2 minus_s, float2 inverse) {
    const float2 q = mul2(y, inverse);
    return fma2(fma2(minus_s, q, y), inverse, q);
}

// Sum over a group of LANES neighbouring lanes.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the CTA.
__device__ __forceinline__ float cta_sum(float v, float *scratch) {
    v = lane_sum<32>(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    return lane_sum<32>(lane < int(blockDim.x >> 5) ? scratch[lane] : 0.f);
}

// A row is cut in units of 8 LANES channels, eight a lane: neighbours where an
// access takes WIDTH (8 or 4) of them; LANES apart where rows are aligned for
// single ones only, so that the lanes of an access are neighbours: 32768 rows of 5119
// in 291 us, 777 x 4099 f16 in 7.3 us (eight neighbours a lane there too: 586 and 22 us).
template <int WIDTH, int LANES>
struct Place {
    static constexpr int kStep = WIDTH == 1 ? LANES : 1;
    int at, n;  // the lane's first channel, and how many of its eight are in the row (<= 0: none)
    Place() = default;
    __device__ __forceinline__ Place(int unit, int lane, int hidden) {
        at = unit * LANES * 8 + (WIDTH == 1 ? lane : lane * 8);
        n = min(8, (hidden - at + kStep - 1) / kStep);
        if (at >= hidden) n = 0;
    }
    template <class T>
    __device__ __forceinline__ void load(const T *row, T (&v)[8]) const {
        const T *p = row + at;
        constexpr int kPer = WIDTH * sizeof(T) < 16 ? WIDTH : 16 / sizeof(T);
        using Piece = std::conditional_t<kPer * sizeof(T) == 16, uint4, std::conditional_t<kPer * sizeof(T) == 8, uint2, T>>;
#pragma unroll
        for (int i = 0; i < 8; i += kPer)
            *reinterpret_cast<Piece *>(v + i) = i < n ? *reinterpret_cast<const Piece *>(p + i * kStep) : Piece{};
    }
    template <class T>
    __device__ __forceinline__ void store(T *row, const T (&v)[8]) const {
        T *p = row + at;
        constexpr int kPer = WIDTH * sizeof(T) < 16 ? WIDTH : 16 / sizeof(T);
        using Piece = std::conditional_t<kPer * sizeof(T) == 16, uint4,
                                         std::conditional_t<kPer * sizeof(T) == 8, uint2,
                                                            std::conditional_t<kPer * sizeof(T) == 4, uint32_t, T>>>;
#pragma unroll
        for (int i = 0; i < 8; i += kPer)
            if (i < n) *reinterpret_cast<Piece *>(p + i * kStep) = *reinterpret_cast<const Piece *>(v + i);
    }
    __device__ __forceinline__ void load_weights(const sq_norm_args &a, float (&w)[8]) const {
        auto from = [&](auto *p) {
            alignas(16) std::remove_const_t<std::remove_pointer_t<decltype(p)>> v[8];
            load(p, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = to_float(v[i]);
        };
        if (a.weight_dtype == SQ_F32) from(static_cast<const float *>(a.weight));
        else if (a.weight_dtype == SQ_BF16) from(static_cast<const __nv_bfloat16 *>(a.weight));
        else from(static_cast<const __half *>(a.weight));
    }
    template <class T>
    __device__ __forceinline__ void round(T *row, const float (&x)[8]) const {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_float<T>(x[i]);
        store(row, v);
    }
    // Eight outputs: in T, or e4m3 with the scale of their 128 channels (every lane of the
    // warp calls; `mine`: there is such a row).
    template <class T>
    __device__ __forceinline__ void put(const sq_norm_args &a, int64_t row, bool mine, const float (&y)[8]) const {
        if (!a.scale) {
            if (mine) round(static_cast<T *>(a.out) + row * a.hidden, y);
            return;
        }
        // Blocks of 128: the eight neighbours of 16 lanes, or 128 / LANES of the eight of the group.
        constexpr int kBlocks = WIDTH == 1 ? LANES / 16 : 1, kEach = 8 / kBlocks;
        alignas(8) uint8_t q[8];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < kEach; ++i) top = max_nan(top, fabsf(y[b * kEach + i]));
#pragma unroll
            for (int o = WIDTH == 1 ? LANES / 2 : 8; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float scale = over_most(max_nan(top, kScaleFloor)), inverse = reciprocal_approx(scale);
            const float minus = inverse == 0.f ? 0.f : -scale;  // an infinite block: its finite values to 0
            const int first = at + b * 128;  // of the block, for its first lane
            if (first % 128 == 0 && first < a.hidden && mine) a.scale[row * ((a.hidden + 127) / 128) + first / 128] = scale;
#pragma unroll
            for (int i = b * kEach; i < (b + 1) * kEach; i += 2)
                *reinterpret_cast<uint16_t *>(q + i) = __nv_cvt_float2_to_fp8x2(
                    quotients(make_float2(y[i], y[i + 1]), make_float2(minus, minus), make_float2(inverse, inverse)),
                    __NV_SATFINITE, __NV_E4M3);
        }
        if (mine) store(static_cast<uint8_t *>(a.out) + row * a.hidden, q);
    }
};

// A row whose squares overflow takes them of h times 2^-80: the largest h is above 2^55 (65536 of
// them overflow no earlier), so nothing that counts underflows; none comes above 2^48, so nothing
// overflows; and eps is nothing beside it.
constexpr float kShrink = 0x1p-80f;

// 1 / sqrt(mean h^2) of such a row, held by groups of LANES lanes of a warp (scratch null) or by the
// CTA.  Passed by value and not inlined: inlined, 32768 x 5119 took 383 us for 291.
template <int CH>
struct Values {
    float h[CH][8];
};
template <int CH, int LANES>
__device__ __noinline__ float large_factor(Values<CH> v, int hidden, float *scratch) {
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float h = v.h[c][i] * kShrink;
            squares += h * h;
        }
    if (scratch) {
        __syncthreads();  // all have read the first sum
        squares = cta_sum(squares, scratch);
    } else {
        squares = lane_sum<LANES>(squares);
    }
    return rsqrtf(squares / float(hidden)) * kShrink;
}
template <int CH, int LANES>
__device__ __forceinline__ float large_factor_of(const float (&h)[CH][8], int hidden, float *scratch) {
    Values<CH> v;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) v.h[c][i] = h[c][i];
    return large_factor<CH, LANES>(v, hidden, scratch);
}

// Short rows: a group of LANES lanes a row, CH units each, the group's next row on
// its way; the weights stay in registers and nothing is shared between warps.
// 100000 bf16 rows of 336 to e4m3: 38 us (a grid of all rows, each warp ending after
// its own, 61 us; two rows a turn, 142 registers, 69 us).
template <class T, int CH, int LANES, int WIDTH>
__global__ void __launch_bounds__(256, CH == 1 ? 4 : 3) norm_lanes_kernel(sq_norm_args a) {
    const int lane = threadIdx.x % LANES;
    const int groups = int(gridDim.x) * (256 / LANES);
    // The row of the warp's first group: the loop's, the same for a warp's lanes.
    const int64_t first = (int64_t(blockIdx.x) * 256 + (threadIdx.x & ~31)) / LANES;
    int64_t row = first + (threadIdx.x & 31) / LANES;
    alignas(16) T x[CH][8], res[CH][8];
    Place<WIDTH, LANES> place[CH];
    float w[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) place[c] = Place<WIDTH, LANES>(c, lane, a.hidden);
    auto fetch = [&](int64_t from) {
        if (from >= a.rows) return;
#pragma unroll
        for (int c = 0; c < CH; ++c) place[c].load(static_cast<const T *>(a.x) + from * a.x_stride, x[c]);
        if (!a.residual) return;
#pragma unroll
        for (int c = 0; c < CH; ++c) place[c].load(static_cast<const T *>(a.residual) + from * a.residual_stride, res[c]);
    };
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[c][i] = from_float<T>(0.f);
            w[c][i] = 1.f;
        }
    fetch(row);
    if (a.weight) {
#pragma unroll
        for (int c = 0; c < CH; ++c) place[c].load_weights(a, w[c]);
    }
    for (int64_t turn = first; turn < a.rows; turn += groups, row += groups) {
        float h[CH][8], squares = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = to_float(x[c][i]);
        if (a.residual) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += to_float(res[c][i]);
        }
        fetch(row + groups);
        const bool mine = row < a.rows;
        if (a.residual && mine) {
#pragma unroll
            for (int c = 0; c < CH; ++c) place[c].round(static_cast<T *>(a.residual_out) + row * a.hidden, h[c]);
        }
        if (a.normalize) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
            squares = lane_sum<LANES>(squares);
            float factor = rsqrtf(squares / float(a.hidden) + a.eps);
            if (__any_sync(0xffffffffu, squares == INFINITY)) {  // in a row of the warp
                const float large = large_factor_of<CH, LANES>(h, a.hidden, nullptr);
                if (squares == INFINITY) factor = large;
            }
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[c][i];
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) place[c].template put<T>(a, row, mine, h[c]);
    }
}

// A CTA a row, each thread with CH steps of 8 values.
template <class T, int CH, int WIDTH>
__global__ void __launch_bounds__(1024) norm_kernel(sq_norm_args a) {
    __shared__ float scratch[32];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float h[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const Place<WIDTH, 32> place(c * warps + warp, lane, a.hidden);
        alignas(16) T x[8], res[8];
        place.load(static_cast<const T *>(a.x) + row * a.x_stride, x);
        if (a.residual) place.load(static_cast<const T *>(a.residual) + row * a.residual_stride, res);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[c][i] = to_float(x[i]);
            if (a.residual) h[c][i] += to_float(res[i]);
        }
    }
    float squares = 0.f, factor = 1.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (a.residual)
            Place<WIDTH, 32>(c * warps + warp, lane, a.hidden).round(static_cast<T *>(a.residual_out) + row * a.hidden, h[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
    }
    if (a.normalize) {
        squares = cta_sum(squares, scratch);
        factor = rsqrtf(squares / float(a.hidden) + a.eps);
        if (squares == INFINITY) factor = large_factor_of<CH, 32>(h, a.hidden, scratch);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const Place<WIDTH, 32> place(c * warps + warp, lane, a.hidden);
        if (a.weight) {
            float w[8];
            place.load_weights(a, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[i];
        }
        place.template put<T>(a, row, true, h[c]);
    }
}

// Many rows of 16-byte aligned pieces: persistent CTAs, kRows rows on their way.
// Each thread copies (cp.async) what it will itself read, so the only barrier of
// a row is its sum's; the weights stay in registers.
constexpr int kRows = 3;

// The CTA's rows first, first + gridDim.x, ... again, those whose squares overflow (or come near),
// after all of them: any branch between the sum and the outputs below costs (65536 x 5120 in 417 to
// 520 us for 385).  Where residual_out is residual's own buffer, it holds the rounded h by now.
template <class T>
__device__ __noinline__ void redo_large(const sq_norm_args &a, int64_t first) {
    __shared__ float scratch[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const bool held = a.residual && a.residual == a.residual_out;
    for (int64_t row = first; row < a.rows; row += gridDim.x) {
        const T *x = held ? static_cast<const T *>(a.residual_out) + row * a.hidden : static_cast<const T *>(a.x) + row * a.x_stride;
        const T *res = a.residual && !held ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
        auto value = [&](int i) { return (to_float(x[i]) + (res ? to_float(res[i]) : 0.f)) * kShrink; };
        __syncthreads();  // the row's outputs are written, and the scratch of the row before is read
        float squares = 0.f;
        for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) squares += value(i) * value(i);
        squares = cta_sum(squares, scratch);
        if (squares < 0x1p-34f) continue;
        const float factor = rsqrtf(squares / float(a.hidden));
        auto normed = [&](int i) {
            const float w = a.weight_dtype == SQ_F32    ? static_cast<const float *>(a.weight)[i]
                            : a.weight_dtype == SQ_BF16 ? to_float(static_cast<const __nv_bfloat16 *>(a.weight)[i])
                                                        : to_float(static_cast<const __half *>(a.weight)[i]);
            return value(i) * factor * w;
        };
        for (int block = warp; block * 128 < a.hidden; block += warps) {
            float y[4], top = 0.f;
            for (int k = 0; k < 4; ++k) {
                const int i = block * 128 + k * 32 + lane;
                y[k] = i < a.hidden ? normed(i) : 0.f;
                top = max_nan(top, fabsf(y[k]));
                if (!a.scale && i < a.hidden) static_cast<T *>(a.out)[row * a.hidden + i] = from_float<T>(y[k]);
            }
            if (!a.scale) continue;
            for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float scale = over_most(max_nan(top, kScaleFloor));
            if (lane == 0) a.scale[row * ((a.hidden + 127) / 128) + block] = scale;
            for (int k = 0; k < 4; ++k) {
                const int i = block * 128 + k * 32 + lane;
                if (i < a.hidden)
                    static_cast<uint8_t *>(a.out)[row * a.hidden + i] = __nv_cvt_float_to_fp8(y[k] / scale, __NV_SATFINITE, __NV_E4M3);
            }
        }
    }
}

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
        if (at < a.hidden) Place<8, 32>(c * (threads / 32) + t / 32, t % 32, a.hidden).load_weights(a, w[c]);
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
    bool large = false;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        fetch(row + int64_t(kRows - 1) * gridDim.x, (stage + kRows - 1) % kRows);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(kRows - 1) : "memory");
        float h[CH][8], squares = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const Place<8, 32> place(c * (threads / 32) + t / 32, t % 32, a.hidden);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = 0.f;
            if (place.n <= 0) continue;
            const T *x = reinterpret_cast<const T *>(slot(stage, 0, c)), *res = reinterpret_cast<const T *>(slot(stage, 1, c));
            alignas(16) T v[8];
            Place<8, 32>(0, 0, 8).load(x, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = to_float(v[i]);
            if (a.residual) {
                Place<8, 32>(0, 0, 8).load(res, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += to_float(v[i]);
                place.round(static_cast<T *>(a.residual_out) + row * a.hidden, h[c]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += h[c][i] * h[c][i];
        }
        squares = cta_sum(squares, scratch[turn]);
        large |= squares == INFINITY;
        const float factor = rsqrtf(squares / float(a.hidden) + a.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * factor * w[c][i];
            Place<8, 32>(c * (threads / 32) + t / 32, t % 32, a.hidden).template put<T>(a, row, true, h[c]);
        }
        stage = stage + 1 == kRows ? 0 : stage + 1;
        turn ^= 1;
    }
    if (large) redo_large<T>(a, blockIdx.x);
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

template <class T, int CH, int LANES, int WIDTH>
cudaError_t launch_lanes(const sq_norm_args &a, cudaStream_t s) {
    const int64_t need = (int64_t(a.rows) * LANES + 255) / 256;
    int64_t room = sms_of(s);
    if (need > room) {
        int each = 0;
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, norm_lanes_kernel<T, CH, LANES, WIDTH>, 256, 0);
        if (e != cudaSuccess) return e;
        room *= each > 0 ? each : 1;
    }
    norm_lanes_kernel<T, CH, LANES, WIDTH><<<unsigned(need < room ? need : room), 256, 0, s>>>(a);
    return cudaGetLastError();
}

template <class T, int WIDTH>
cudaError_t launch_width(const sq_norm_args &a, cudaStream_t s) {
    const int steps = (a.hidden + 7) / 8;
    if (steps <= 16) return launch_lanes<T, 1, 16, WIDTH>(a, s);
    if (steps <= 32) return launch_lanes<T, 1, 32, WIDTH>(a, s);
    if (steps <= 64) return launch_lanes<T, 2, 32, WIDTH>(a, s);
    // Rows on their way while others are worked on, once each resident CTA has several.
    if (WIDTH == 8 && a.normalize && a.rows >= 2048 && steps <= 2048) {
        const int ch = steps <= 1024 ? 2 : 4, threads = ((steps + ch - 1) / ch + 31) / 32 * 32;
        const int bytes = kRows * 2 * ch * threads * 8 * int(sizeof(T));
        if (bytes <= 200 * 1024)
            return ch == 2 ? launch_rows<T, 2>(a, threads, bytes, s) : launch_rows<T, 4>(a, threads, bytes, s);
    }
    // The CTA a row: few rows spread over many threads, many rows two or more steps a thread.
    int ch = a.rows < 592 ? 1 : 2;
    while (ch < 8 && steps > 1024 * ch) ch *= 2;
    const int threads = ((steps + ch - 1) / ch + 31) / 32 * 32;
    const unsigned grid = unsigned(a.rows);
    switch (ch) {
        case 1: norm_kernel<T, 1, WIDTH><<<grid, threads, 0, s>>>(a); break;
        case 2: norm_kernel<T, 2, WIDTH><<<grid, threads, 0, s>>>(a); break;
        case 4: norm_kernel<T, 4, WIDTH><<<grid, threads, 0, s>>>(a); break;
        default: norm_kernel<T, 8, WIDTH><<<grid, threads, 0, s>>>(a); break;
    }
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
    return fits(8) ? launch_width<T, 8>(a, s) : fits(4) ? launch_width<T, 4>(a, s) : launch_width<T, 1>(a, s);
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
