// Short causal convolution of recurrent layers, one filter of 2 to 4 taps a
// channel, for prompts (concatenated sequences) and for single tokens.
//
//   y[t, d] = act(bias[d] + sum_j w[d, j] x[t - W + 1 + j, d])
//
// Inputs before a sequence's first token come from its state row
// [channels, W - 1] (oldest first), or are zero; the row after the call holds
// the last W - 1 inputs.  Products, sum and activation are fp32; y and the
// state are rounded to, or copied in, the input's type.
//
// Bound by bytes: x read once, y written once, the W - 1 inputs before a token
// kept in registers.  A thread takes eight channels (16 bytes of a 16-bit row)
// and walks a strip of tokens; strips overlap by their W - 1 leading inputs.
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kConvThreads = 128;

// Strip `index` of the concatenated sequences: sequence n owns the indices from
// cu[n] / strip + n on, at least as many as its strips, so a strip finds its
// sequence by bisection and strip 0 exists for an empty sequence too.
__device__ __forceinline__ int find_sequence(const int32_t *cu, int seqs, int tokens, int strip, int64_t index) {
    int lo = 0, hi = seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (max(0, min(cu[mid], tokens)) / strip + int64_t(mid) <= index) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// State row of request n: n itself, or slots[n].  -1: a padded request (slot
// <= 0) or, flagged in status, a slot outside the pool.
__device__ __forceinline__ int64_t state_row(const int64_t *slots, int n, int64_t num_slots, int32_t *status) {
    if (!slots) return n;
    const int64_t slot = slots[n];
    if (slot >= num_slots) {
        flag(status, SQ_STATUS_SLOT_RANGE);
        return -1;
    }
    return slot <= 0 ? -1 : slot;
}

template <class T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&x)[VEC]) {
    if (VEC == 8) load8(p, true, 8, *reinterpret_cast<float(*)[8]>(&x));
    else x[0] = to_float(*p);
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[VEC]) {
    if (VEC == 8) store8(p, true, 8, *reinterpret_cast<const float(*)[8]>(&x));
    else *p = from_float<T>(x[0]);
}

template <class T, int VEC, int W>
__global__ void __launch_bounds__(kConvThreads) conv_kernel(sq_conv_args a, int strip) {
    const int d0 = (blockIdx.y * kConvThreads + threadIdx.x) * VEC;
    if (d0 >= a.channels) return;
    const int n = find_sequence(a.cu_seqlens, a.num_seqs, a.tokens, strip, blockIdx.x);
    const int begin = max(0, min(a.cu_seqlens[n], a.tokens));
    const int end = max(begin, min(a.cu_seqlens[n + 1], a.tokens));
    const int64_t part = blockIdx.x - (begin / strip + int64_t(n));  // strip of the sequence
    if (part < 0 || (part > 0 && part * strip >= end - begin)) return;
    const int t0 = begin + int(part) * strip, t1 = min(end, t0 + strip);
    const int64_t row = state_row(a.slots, n, a.num_slots, a.status);
    T *y = static_cast<T *>(a.y) + d0;
    float zero[VEC] = {};
    if (row < 0) {
        for (int t = t0; t < t1; ++t) store_vec<T, VEC>(y + int64_t(t) * a.channels, zero);
        return;
    }
    const T *x = static_cast<const T *>(a.x) + d0;
    const T *old = a.initial_state ? static_cast<const T *>(a.initial_state) + (row * a.channels + d0) * (W - 1) : nullptr;
    float w[VEC][W], bias[VEC], kept[W - 1][VEC];  // kept[j]: input W - 1 - j tokens back
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        bias[i] = a.bias ? a.bias[d0 + i] : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = a.weight[int64_t(d0 + i) * W + j];
    }
    // Input of token t of the sequence, t < begin from the state.
    auto input = [&](int64_t t, float(&v)[VEC]) {
        if (t >= begin) {
            load_vec<T, VEC>(x + t * a.x_stride, v);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = old ? to_float(old[i * (W - 1) + int(t - begin) + W - 1]) : 0.f;
        }
    };
#pragma unroll
    for (int j = 0; j < W - 1; ++j) input(int64_t(t0) - (W - 1) + j, kept[j]);
    float last[W - 1][VEC];
    if (part == 0 && a.final_state) {  // read before any write: the two states may be one buffer
#pragma unroll
        for (int j = 0; j < W - 1; ++j) input(int64_t(end) - (W - 1) + j, last[j]);
    }
#pragma unroll 4
    for (int t = t0; t < t1; ++t) {
        float now[VEC], out[VEC];
        load_vec<T, VEC>(x + int64_t(t) * a.x_stride, now);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float s = bias[i];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) s = fmaf(w[i][j], kept[j][i], s);
            s = fmaf(w[i][W - 1], now[i], s);
            out[i] = a.silu ? silu(s) : s;
        }
        store_vec<T, VEC>(y + int64_t(t) * a.channels, out);
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) kept[j][i] = kept[j + 1][i];
#pragma unroll
        for (int i = 0; i < VEC; ++i) kept[W - 2][i] = now[i];
    }
    if (part == 0 && a.final_state) {
        T *fin = static_cast<T *>(a.final_state) + (row * a.channels + d0) * (W - 1);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
#pragma unroll
            for (int j = 0; j < W - 1; ++j) fin[i * (W - 1) + j] = from_float<T>(last[j][i]);
    }
}

// One token of each request: the state row shifts by one input.
template <class T, int VEC, int W>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(sq_conv_args a) {
    const int d0 = (blockIdx.y * kConvThreads + threadIdx.x) * VEC;
    if (d0 >= a.channels) return;
    const int n = blockIdx.x;
    const int64_t row = state_row(a.slots, n, a.num_slots, a.status);
    T *y = static_cast<T *>(a.y) + int64_t(n) * a.channels + d0;
    float now[VEC], out[VEC] = {};
    if (row < 0) {
        store_vec<T, VEC>(y, out);
        return;
    }
    T *state = static_cast<T *>(a.final_state) + (row * a.channels + d0) * (W - 1);
    load_vec<T, VEC>(static_cast<const T *>(a.x) + int64_t(n) * a.x_stride + d0, now);
    T kept[VEC * (W - 1)];
#pragma unroll
    for (int i = 0; i < VEC * (W - 1); ++i) kept[i] = state[i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float s = a.bias ? a.bias[d0 + i] : 0.f;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) s = fmaf(a.weight[int64_t(d0 + i) * W + j], to_float(kept[i * (W - 1) + j]), s);
        s = fmaf(a.weight[int64_t(d0 + i) * W + W - 1], now[i], s);
        out[i] = a.silu ? silu(s) : s;
    }
    store_vec<T, VEC>(y, out);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
        for (int j = 0; j < W - 1; ++j) state[i * (W - 1) + j] = j + 1 < W - 1 ? kept[i * (W - 1) + j + 1] : from_float<T>(now[i]);
}

template <class T, int VEC, int W>
cudaError_t launch_conv_as(const sq_conv_args &a, bool step, cudaStream_t s) {
    const unsigned columns = unsigned((int64_t(a.channels) + kConvThreads * VEC - 1) / (kConvThreads * VEC));
    if (step) {
        conv_step_kernel<T, VEC, W><<<dim3(unsigned(a.num_seqs), columns), kConvThreads, 0, s>>>(a);
        return cudaGetLastError();
    }
    // Strips of 64 tokens; shorter ones while the grid would leave SMs idle.
    int strip = 64;
    while (strip > 8 && int64_t(a.tokens / strip + a.num_seqs) * columns < 148 * 8) strip /= 2;
    conv_kernel<T, VEC, W><<<dim3(unsigned(a.tokens / strip + a.num_seqs), columns), kConvThreads, 0, s>>>(a, strip);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_conv(const sq_conv_args &a, bool step, cudaStream_t s) {
    const bool vec = a.channels % 8 == 0 && aligned16(a.x) && aligned16(a.y) && a.x_stride * int64_t(sizeof(T)) % 16 == 0 &&
                     a.channels * int64_t(sizeof(T)) % 16 == 0;
    switch (a.taps) {
        case 2: return vec ? launch_conv_as<T, 8, 2>(a, step, s) : launch_conv_as<T, 1, 2>(a, step, s);
        case 3: return vec ? launch_conv_as<T, 8, 3>(a, step, s) : launch_conv_as<T, 1, 3>(a, step, s);
        default: return vec ? launch_conv_as<T, 8, 4>(a, step, s) : launch_conv_as<T, 1, 4>(a, step, s);
    }
}

int32_t conv_entry(const sq_conv_args *args, bool step, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_conv_args &a = *args;
    if (a.tokens < 0 || a.num_seqs < 0 || a.channels < 1 || (a.slots && a.num_slots < 1)) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.taps < 2 || a.taps > 4) return SQ_ERR_UNSUPPORTED;
    if (a.x_stride < 0) return SQ_ERR_SHAPE;
    if (a.channels > (1 << 22)) return SQ_ERR_UNSUPPORTED;
    if (a.num_seqs == 0) return SQ_OK;
    if (!a.weight || (a.tokens > 0 && (!a.x || !a.y))) return SQ_ERR_ARGUMENT;
    if (step ? !a.final_state : !a.cu_seqlens) return SQ_ERR_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? launch_conv<float>(a, step, s)
                          : a.dtype == SQ_BF16 ? launch_conv<__nv_bfloat16>(a, step, s)
                                               : launch_conv<__half>(a, step, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_causal_conv(const sq_conv_args *args, sq_stream_t stream) { return sq::conv_entry(args, false, stream); }

extern "C" int32_t sq_causal_conv_step(const sq_conv_args *args, sq_stream_t stream) { return sq::conv_entry(args, true, stream); }
