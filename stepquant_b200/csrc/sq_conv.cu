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
// kept in registers.  A thread takes four channels (8 bytes of a 16-bit row)
// and walks a strip of tokens, eight tokens in flight while the eight before are
// worked on; strips overlap by their W - 1 leading inputs.  Measured at 8192 bf16
// channels: 32768 tokens in 181 us (5.9 TB/s, 0.92 of the measured copy); eight
// channels a thread 431 us (loads held behind stores, half the threads), a branch
// between the tokens of a batch 218 us.  One token of 256 requests 8.6 us (4 TB/s).
// Rows aligned for two channels or one take them so, with more instructions a byte:
// 8190 channels 232 us (singly 312), 8191 in 297 us; one token 8.7 and 11.6 us.
#include <type_traits>

#include "sq_rows.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kConvThreads = 128;
constexpr unsigned kGridRows = 32768;  // requests along a grid's second axis, the rest along its third

// N values of VEC channels (a token's, or a state row's), by accesses of VEC channels, at most 16 bytes.
template <class T, int N, int VEC>
struct Run {
    static constexpr int kPiece = VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16;
    using Piece = std::conditional_t<kPiece == 16, uint4, std::conditional_t<kPiece == 8, uint2, uint32_t>>;
    alignas(16) T v[N];
    __device__ __forceinline__ void load(const T *p) {
        if (VEC > 1) {
#pragma unroll
            for (int i = 0; i < int(N * sizeof(T) / kPiece); ++i) reinterpret_cast<Piece *>(v)[i] = reinterpret_cast<const Piece *>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if (VEC > 1) {
#pragma unroll
            for (int i = 0; i < int(N * sizeof(T) / kPiece); ++i) reinterpret_cast<Piece *>(p)[i] = reinterpret_cast<const Piece *>(v)[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = v[i];
        }
    }
};

// bias and weights of VEC channels, [channel][tap].
template <int VEC, int W>
struct Filter {
    float w[VEC * W], bias[VEC];
    __device__ __forceinline__ Filter(const sq_conv_args &a, int d0) {
        Run<float, VEC * W, VEC> r;
        r.load(a.weight + int64_t(d0) * W);
        Run<float, VEC, VEC> s;
        if (a.bias) s.load(a.bias + d0);
#pragma unroll
        for (int i = 0; i < VEC * W; ++i) w[i] = r.v[i];
#pragma unroll
        for (int i = 0; i < VEC; ++i) bias[i] = a.bias ? s.v[i] : 0.f;
    }
};

// The CTAs past `strips` clear the tokens of no sequence.
template <class T, int VEC, int W, bool SILU>
__global__ void __launch_bounds__(kConvThreads) conv_kernel(sq_conv_args a, int strip, unsigned strips) {
    using Token = Run<T, VEC, VEC>;
    constexpr int BATCH = 8;  // tokens in flight a thread, while the batch before is worked on
    if (blockIdx.x >= strips) {
        clear_outside(a.y, int64_t(a.channels) * sizeof(T), a.cu_seqlens, a.num_seqs, a.tokens,
                      (blockIdx.x - strips) * gridDim.y + blockIdx.y, (gridDim.x - strips) * gridDim.y);
        return;
    }
    const int d0 = (blockIdx.y * kConvThreads + threadIdx.x) * VEC;
    if (d0 >= a.channels) return;
    const int n = sequence_of(a.cu_seqlens, a.num_seqs, a.tokens, strip, blockIdx.x);
    const int2 seq = sequence_range(a.cu_seqlens, n, a.tokens);
    const int begin = seq.x, end = seq.y;
    const int64_t part = blockIdx.x - (begin / strip + int64_t(n));  // strip of the sequence
    if (part < 0 || (part > 0 && part * strip >= end - begin)) return;
    const int t0 = begin + int(part) * strip, t1 = min(end, t0 + strip);
    const int64_t row = state_row(a.slots, n, a.num_slots, a.status);
    T *y = static_cast<T *>(a.y) + d0;
    if (row < 0) {
        Token zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.v[i] = from_float<T>(0.f);
        for (int t = t0; t < t1; ++t) zero.store(y + int64_t(t) * a.channels);
        return;
    }
    const T *x = static_cast<const T *>(a.x) + d0;
    const int64_t state = (row * a.channels + d0) * (W - 1);
    const T *old = a.initial_state ? static_cast<const T *>(a.initial_state) + state : nullptr;
    Token next[BATCH], now[BATCH];
    auto fetch = [&](int t) {
        const T *from = x + int64_t(t) * a.x_stride;
        if (t + BATCH <= t1) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j, from += a.x_stride) next[j].load(from);
        } else {
#pragma unroll
            for (int j = 0; j < BATCH; ++j, from += a.x_stride)
                if (t + j < t1) next[j].load(from);
        }
    };
    fetch(t0);
    const Filter<VEC, W> f(a, d0);
    // Input of token t of the sequence, t < begin from the state.
    auto input = [&](int64_t t, Token &v) {
        if (t >= begin) {
            v.load(x + t * a.x_stride);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v.v[i] = old ? old[i * (W - 1) + int(t - begin) + W - 1] : from_float<T>(0.f);
        }
    };
    float kept[W - 1][VEC];  // kept[j]: input W - 1 - j tokens back
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        Token v;
        input(int64_t(t0) - (W - 1) + j, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) kept[j][i] = to_float(v.v[i]);
    }
    if (part == 0 && a.final_state) {  // the strip that reads the state writes it, after reading: they may be one buffer
        Run<T, VEC * (W - 1), VEC> fin;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            Token v;
            input(int64_t(end) - (W - 1) + j, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) fin.v[i * (W - 1) + j] = v.v[i];
        }
        fin.store(static_cast<T *>(a.final_state) + state);
    }
    T *to = y + int64_t(t0) * a.channels;
    auto token = [&](const Token &in) {
        Token out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float x_t = to_float(in.v[i]);
            float s = f.bias[i];
#pragma unroll
            for (int k = 0; k < W - 1; ++k) s = fmaf(f.w[i * W + k], kept[k][i], s);
            s = fmaf(f.w[i * W + W - 1], x_t, s);
            out.v[i] = from_float<T>(SILU ? silu(s) : s);
#pragma unroll
            for (int k = 0; k + 1 < W - 1; ++k) kept[k][i] = kept[k + 1][i];
            kept[W - 2][i] = x_t;
        }
        out.store(to);
        to += a.channels;
    };
    for (int t = t0; t < t1; t += BATCH) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) now[j] = next[j];
        fetch(t + BATCH);
        if (t + BATCH <= t1) {  // no branch between the tokens of a whole batch
#pragma unroll
            for (int j = 0; j < BATCH; ++j) token(now[j]);
        } else {
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (t + j < t1) token(now[j]);
        }
    }
}

// One token of each request: the state row shifts by one input.
template <class T, int VEC, int W>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(sq_conv_args a) {
    // Neighbouring CTAs take neighbouring channels of a request.
    const int n = blockIdx.z * kGridRows + blockIdx.y, d0 = (blockIdx.x * kConvThreads + threadIdx.x) * VEC;
    if (d0 >= a.channels || n >= a.num_seqs) return;
    const int64_t row = state_row(a.slots, n, a.num_slots, a.status);
    Run<T, VEC, VEC> in, out;
    T *y = static_cast<T *>(a.y) + int64_t(n) * a.channels + d0;
    if (row < 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out.v[i] = from_float<T>(0.f);
        out.store(y);
        return;
    }
    T *state = static_cast<T *>(a.final_state) + (row * a.channels + d0) * (W - 1);
    Run<T, VEC * (W - 1), VEC> kept;
    in.load(static_cast<const T *>(a.x) + int64_t(n) * a.x_stride + d0);
    kept.load(state);
    const Filter<VEC, W> f(a, d0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float s = f.bias[i];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) s = fmaf(f.w[i * W + j], to_float(kept.v[i * (W - 1) + j]), s);
        s = fmaf(f.w[i * W + W - 1], to_float(in.v[i]), s);
        out.v[i] = from_float<T>(a.silu ? silu(s) : s);
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j) kept.v[i * (W - 1) + j] = kept.v[i * (W - 1) + j + 1];
        kept.v[i * (W - 1) + W - 2] = in.v[i];
    }
    out.store(y);
    kept.store(state);
}

template <class T, int VEC, int W>
cudaError_t launch_conv_as(const sq_conv_args &a, bool step, cudaStream_t s) {
    const unsigned columns = unsigned((int64_t(a.channels) + kConvThreads * VEC - 1) / (kConvThreads * VEC));
    if (step) {
        const unsigned rows = unsigned(a.num_seqs);
        const dim3 grid(columns, rows < kGridRows ? rows : kGridRows, (rows + kGridRows - 1) / kGridRows);
        conv_step_kernel<T, VEC, W><<<grid, kConvThreads, 0, s>>>(a);
        return cudaGetLastError();
    }
    // Strips of 64 tokens; shorter ones while the grid would leave SMs idle (of a whole GPU's 148:
    // a stream of fewer takes the same strips).
    int strip = 64;
    while (strip > 8 && int64_t(a.tokens / strip + a.num_seqs) * columns < 148 * 8) strip /= 2;
    const unsigned strips = unsigned(a.tokens / strip + a.num_seqs);
    const dim3 grid(strips + (147 + columns) / columns, columns);
    if (a.silu) conv_kernel<T, VEC, W, true><<<grid, kConvThreads, 0, s>>>(a, strip, strips);
    else conv_kernel<T, VEC, W, false><<<grid, kConvThreads, 0, s>>>(a, strip, strips);
    return cudaGetLastError();
}

template <class T, int VEC>
cudaError_t launch_taps(const sq_conv_args &a, bool step, cudaStream_t s) {
    switch (a.taps) {
        case 2: return launch_conv_as<T, VEC, 2>(a, step, s);
        case 3: return launch_conv_as<T, VEC, 3>(a, step, s);
        default: return launch_conv_as<T, VEC, 4>(a, step, s);
    }
}

template <class T>
cudaError_t launch_conv(const sq_conv_args &a, bool step, cudaStream_t s) {
    auto fits = [&](int n) {  // rows of pieces of n channels
        auto on = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0; };
        return a.channels % n == 0 && a.x_stride % n == 0 && on(a.x) && on(a.y) && on(a.initial_state) && on(a.final_state) &&
               aligned16(a.weight) && aligned16(a.bias);
    };
    return fits(4) ? launch_taps<T, 4>(a, step, s) : fits(2) ? launch_taps<T, 2>(a, step, s) : launch_taps<T, 1>(a, step, s);
}

int32_t conv_entry(const sq_conv_args *args, bool step, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_conv_args &a = *args;
    if (a.tokens < 0 || a.num_seqs < 0 || a.channels < 1 || (a.slots && a.num_slots < 1)) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.taps < 2 || a.taps > 4) return SQ_ERR_UNSUPPORTED;
    if (a.x_stride < 0) return SQ_ERR_SHAPE;
    if (a.channels > (1 << 22) || a.num_seqs > (1 << 30) || a.tokens > kMostTokens) return SQ_ERR_UNSUPPORTED;
    if (a.num_seqs == 0) return SQ_OK;
    if (!a.weight || (a.tokens > 0 && (!a.x || !a.y))) return SQ_ERR_ARGUMENT;
    if (step ? !a.final_state : !a.cu_seqlens) return SQ_ERR_ARGUMENT;
    if (!a.slots && a.num_slots > 0 && a.num_slots < a.num_seqs) return SQ_ERR_CAPACITY;  // state row n of a smaller pool
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
