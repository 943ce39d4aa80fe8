// Rotary positions: pairs of channels turned by position * frequency.
//
// A CTA takes up to 16 tokens: the sines and cosines of their angles go to shared
// memory once and serve all heads (two multiplications and two fused ones a pair
// beside them), so the bytes of x and out bound it.
#include "sq_kv.cuh"
#include "sq_rows.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kRotaryThreads = 256;

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

template <class T, int VEC>
struct Piece {
    T x[VEC];
    __device__ __forceinline__ void load(const T *p) {
        using R = typename Raw<VEC * sizeof(T)>::type;
        *reinterpret_cast<R *>(x) = *reinterpret_cast<const R *>(p);
    }
    __device__ __forceinline__ void store(T *p) const {
        using R = typename Raw<VEC * sizeof(T)>::type;
        *reinterpret_cast<R *>(p) = *reinterpret_cast<const R *>(x);
    }
};

// Units of a head: pieces of VEC channels; `turned_units` of them are rotated, each with its partner piece
// VEC channels of the other half, or (interleaved) pairs of its own.
template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, 4) rotary_kernel(sq_rotary_args a, int per_cta, int turned_units, int units, bool copy) {
    extern __shared__ float2 table[];  // [per_cta][turned / 2] (cos, sin), times the magnitude
    const int half = a.turned / 2;
    const int64_t first = int64_t(blockIdx.x) * per_cta;
    const int count = int(min(int64_t(per_cta), a.tokens - first));
    for (int i = threadIdx.x; i < count * half; i += kRotaryThreads) {
        const int t = i / half, f = i - t * half;
        const int64_t phase = phase_of(position_at(a.positions, a.position_dtype, first + t), a.frequencies[f]);
        float sin, cos;
        sincospif(float(int32_t(phase >> 32)) * 0x1p-31f, &sin, &cos);
        table[i] = make_float2(a.magnitude * cos, a.inverse ? -a.magnitude * sin : a.magnitude * sin);
    }
    __syncthreads();
    const int live = copy ? units : turned_units;
    const int slots = a.heads * live;
    // Threads are [token][slot] where a token's slots are fewer than them.
    const int lanes = slots < kRotaryThreads ? kRotaryThreads / max(slots, 1) : 1;
    const int lane = slots < kRotaryThreads ? int(threadIdx.x) / max(slots, 1) : 0;
    if (lane >= lanes) return;
    for (int slot = int(threadIdx.x) - lane * slots; slot < slots; slot += kRotaryThreads) {
        const int head = slot / live, unit = slot - head * live;
        const T *x = static_cast<const T *>(a.x) + head * a.x_head_stride;
        T *out = static_cast<T *>(a.out) + head * a.out_head_stride;
        // Two tokens are read before either is written (out may be x, so the compiler would not).
        constexpr int K = 2;
        const int64_t x_step = lanes * a.x_stride, out_step = lanes * a.out_stride;
        x += (first + lane) * a.x_stride;
        out += (first + lane) * a.out_stride;
        if (unit >= turned_units) {
            const int c = a.turned + (unit - turned_units) * VEC;
            x += c;
            out += c;
            for (int t = lane; t < count; t += K * lanes, x += K * x_step, out += K * out_step) {
                Piece<T, VEC> p[K];
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (t + k * lanes < count) p[k].load(x + k * x_step);
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (t + k * lanes < count) p[k].store(out + k * out_step);
            }
        } else if (INTERLEAVED) {
            constexpr int W = VEC < 2 ? 2 : VEC, S = VEC < 2 ? 1 : VEC;  // channels of a unit, and of an access
            x += unit * W;
            out += unit * W;
            for (int t = lane; t < count; t += K * lanes, x += K * x_step, out += K * out_step) {
                Piece<T, S> p[K][W / S];
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < W / S; ++i)
                        if (t + k * lanes < count) p[k][i].load(x + k * x_step + i * S);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (t + k * lanes >= count) break;
                    const float2 *cs = table + (t + k * lanes) * half + unit * (W / 2);
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        const float2 z = cs[i / 2];
                        T &e = p[k][i / S].x[i % S], &o = p[k][(i + 1) / S].x[(i + 1) % S];
                        const float u = to_float(e), v = to_float(o);
                        e = from_float<T>(u * z.x - v * z.y);
                        o = from_float<T>(u * z.y + v * z.x);
                    }
#pragma unroll
                    for (int i = 0; i < W / S; ++i) p[k][i].store(out + k * out_step + i * S);
                }
            }
        } else {
            const int c = unit * VEC;
            x += c;
            out += c;
            for (int t = lane; t < count; t += K * lanes, x += K * x_step, out += K * out_step) {
                Piece<T, VEC> p[K], q[K];
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (t + k * lanes < count) {
                        p[k].load(x + k * x_step);
                        q[k].load(x + k * x_step + half);
                    }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (t + k * lanes >= count) break;
                    const float2 *cs = table + (t + k * lanes) * half + c;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float2 z = cs[i];
                        const float u = to_float(p[k].x[i]), v = to_float(q[k].x[i]);
                        p[k].x[i] = from_float<T>(u * z.x - v * z.y);
                        q[k].x[i] = from_float<T>(u * z.y + v * z.x);
                    }
                    p[k].store(out + k * out_step);
                    q[k].store(out + k * out_step + half);
                }
            }
        }
    }
}

template <class T, int VEC>
cudaError_t launch_rotary(const sq_rotary_args &a, cudaStream_t s) {
    // Fewer tokens a CTA while the grid would leave SMs idle.
    int per_cta = 16;
    while (per_cta > 1 && (int64_t(a.tokens) + per_cta - 1) / per_cta < 148 * 4) per_cta /= 2;
    const bool copy = a.x != a.out || a.x_stride != a.out_stride || a.x_head_stride != a.out_head_stride;
    const int wide = VEC < 2 && a.interleaved ? 2 : VEC;
    const int turned_units = a.interleaved ? a.turned / wide : a.turned / 2 / VEC;
    const int units = turned_units + (a.dim - a.turned) / VEC;
    const unsigned grid = unsigned((int64_t(a.tokens) + per_cta - 1) / per_cta);
    const size_t shared = size_t(per_cta) * (a.turned / 2) * sizeof(float2);
    auto kernel = a.interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>;
    if (shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
        if (e != cudaSuccess) return e;
    }
    kernel<<<grid, kRotaryThreads, shared, s>>>(a, per_cta, turned_units, units, copy);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_rotary(const sq_rotary_args &a, cudaStream_t s) {
    auto fits = [&](int n) {  // pieces of n channels
        auto on = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0; };
        const int span = a.interleaved ? a.turned : a.turned / 2;
        return span % n == 0 && a.dim % n == 0 && (a.dim - a.turned) % n == 0 && on(a.x) && on(a.out) && a.x_stride % n == 0 &&
               a.x_head_stride % n == 0 && a.out_stride % n == 0 && a.out_head_stride % n == 0;
    };
    constexpr int kWide = 16 / sizeof(T);
    return fits(kWide) ? launch_rotary<T, kWide>(a, s) : fits(2) ? launch_rotary<T, 2>(a, s) : launch_rotary<T, 1>(a, s);
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_rotary(const sq_rotary_args *args, sq_stream_t stream) {
    using namespace sq;
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_rotary_args &a = *args;
    if (a.tokens < 0 || a.heads < 0 || a.dim < 1 || a.turned < 0 || a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (!(fabsf(a.magnitude) < INFINITY)) return SQ_ERR_ARGUMENT;
    if (a.turned % 2 || a.turned > a.dim || a.x_stride < 0 || a.x_head_stride < 0 || a.out_stride < 0 || a.out_head_stride < 0)
        return SQ_ERR_SHAPE;
    if (a.dim > 1024 || a.heads > (1 << 20) || a.tokens > kMostTokens) return SQ_ERR_UNSUPPORTED;
    if (a.tokens == 0 || a.heads == 0) return SQ_OK;
    if (!a.x || !a.out || (a.turned && (!a.positions || !a.frequencies))) return SQ_ERR_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? launch_rotary<float>(a, s)
                          : a.dtype == SQ_BF16 ? launch_rotary<__nv_bfloat16>(a, s)
                                               : launch_rotary<__half>(a, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}
