// Selective state space scan, for prompts (concatenated sequences) and for
// single tokens.  Channel d of group G = d / (channels / groups), state n:
//
//   dt' = softplus(dt + dt_bias)
//   h[d, n] <- exp(dt' A[d, n]) h[d, n] + dt' u B[G, n]
//   y[d] = (sum_n C[G, n] h[d, n] + D[d] u) silu(z)
//
// h, A and every intermediate are fp32; y is rounded once to the input's type.
//
// Prompts: four states a lane, N / 4 lanes a channel; a CTA of 128 lanes walks
// its channels through the sequence in tiles of 32 tokens.  Per tile the CTA
// forms dt', dt' u once per (token, channel) in shared memory, the lanes run
// the recurrence in registers, and the outputs leave through shared memory.
// Bound by the special function unit: one exponential per (token, channel,
// state) at 16 a clock and SM.
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kScanThreads = 128;
constexpr int kTile = 32;     // tokens of a tile
constexpr int kPerLane = 4;   // states of a lane
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// expf, not its fast form: far below zero softplus is the exponential, and the
// step size scales every input of the state.
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

__device__ __forceinline__ int64_t scan_row(const int64_t *slots, int n, int64_t num_slots, int32_t *status) {
    if (!slots) return n;
    const int64_t slot = slots[n];
    if (slot >= num_slots) {
        flag(status, SQ_STATUS_SLOT_RANGE);
        return -1;
    }
    return slot <= 0 ? -1 : slot;
}

// A lane's four entries of a state or A row (16-byte aligned: N is a multiple of 4).
__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

template <class T, int N>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(sq_scan_args a) {
    constexpr int P = N / kPerLane;              // lanes of a channel
    constexpr int CH = kScanThreads / P;         // channels of the CTA
    __shared__ float2 step[kTile][CH];           // dt', dt' u; then y in .x
    __shared__ float4 bs[kTile][P], cs[kTile][P];
    const int tid = threadIdx.x, lane = tid % P, ch = tid / P;
    const int per = a.channels / a.groups, tiles = (per + CH - 1) / CH;  // CTAs of a group
    const int group = blockIdx.y / tiles, first = (blockIdx.y - group * tiles) * CH;
    const int live = min(CH, per - first), d0 = group * per + first;
    const int n = blockIdx.x;
    const int begin = max(0, min(a.cu_seqlens[n], a.tokens));
    const int end = max(begin, min(a.cu_seqlens[n + 1], a.tokens));
    const int64_t row = scan_row(a.slots, n, a.num_slots, a.status);
    T *y = static_cast<T *>(a.y) + d0;
    if (row < 0) {
        for (int64_t i = tid; i < (end - begin) * int64_t(CH); i += kScanThreads)
            if (i % CH < live) y[(begin + i / CH) * a.channels + i % CH] = from_float<T>(0.f);
        return;
    }
    const T *u = static_cast<const T *>(a.u) + d0, *dt = static_cast<const T *>(a.dt) + d0;
    const T *z = a.z ? static_cast<const T *>(a.z) + d0 : nullptr;
    const T *b = static_cast<const T *>(a.b) + group * N, *c = static_cast<const T *>(a.c) + group * N;
    const int mine = min(ch, live - 1);  // lanes past the group's channels follow its last
    float A[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    load4(a.a + int64_t(d0 + mine) * N + lane * 4, A);
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] *= kLog2e;
    const int64_t at = (row * a.channels + d0 + mine) * N + lane * 4;
    if (a.initial_state) load4(a.initial_state + at, h);
    for (int t0 = begin; t0 < end; t0 += kTile) {
        const int count = min(kTile, end - t0);
        for (int i = tid; i < count * CH; i += kScanThreads) {
            const int t = i / CH, k = min(i % CH, live - 1);
            const float d = to_float(dt[(t0 + t) * a.dt_stride + k]) + (a.dt_bias ? a.dt_bias[d0 + k] : 0.f);
            const float s = a.softplus ? softplus(d) : d;
            step[t][i % CH] = make_float2(s, s * to_float(u[(t0 + t) * a.u_stride + k]));
        }
        for (int i = tid; i < count * N; i += kScanThreads) {
            const int t = i / N, k = i % N;
            reinterpret_cast<float *>(bs[t])[k] = to_float(b[(t0 + t) * a.b_stride + k]);
            reinterpret_cast<float *>(cs[t])[k] = to_float(c[(t0 + t) * a.c_stride + k]);
        }
        __syncthreads();
        for (int t = 0; t < count; ++t) {
            const float2 s = step[t][ch];
            const float4 bv = bs[t][lane], cv = cs[t][lane];
            const float bb[4] = {bv.x, bv.y, bv.z, bv.w}, cc[4] = {cv.x, cv.y, cv.z, cv.w};
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = fmaf(exp2_approx(s.x * A[i]), h[i], s.y * bb[i]);
                sum = fmaf(cc[i], h[i], sum);
            }
#pragma unroll
            for (int o = P / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) step[t][ch].x = sum;
        }
        __syncthreads();
        for (int i = tid; i < count * CH; i += kScanThreads) {
            const int t = i / CH, k = i % CH;
            if (k >= live) continue;
            const int64_t tok = t0 + t;
            float out = step[t][k].x;
            if (a.d) out = fmaf(a.d[d0 + k], to_float(u[tok * a.u_stride + k]), out);
            if (z) out *= silu(to_float(z[tok * a.z_stride + k]));
            y[tok * a.channels + k] = from_float<T>(out);
        }
        __syncthreads();
    }
    if (a.final_state && ch < live) *reinterpret_cast<float4 *>(a.final_state + at) = make_float4(h[0], h[1], h[2], h[3]);
}

// One token of each request: N / 4 lanes a channel, the state read and written once.
template <class T, int N>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(sq_scan_args a) {
    constexpr int P = N / kPerLane;
    const int lane = threadIdx.x % P, n = blockIdx.x;
    const int d = (blockIdx.y * kScanThreads + threadIdx.x) / P;
    const bool live = d < a.channels;
    const int k = live ? d : a.channels - 1, group = k / (a.channels / a.groups);
    const int64_t row = scan_row(a.slots, n, a.num_slots, a.status);
    T *y = static_cast<T *>(a.y) + int64_t(n) * a.channels;
    if (row < 0) {
        if (live && lane == 0) y[d] = from_float<T>(0.f);
        return;
    }
    float *state = a.final_state + (row * a.channels + k) * N + lane * 4;
    float A[4], h[4];
    load4(a.a + int64_t(k) * N + lane * 4, A);
    load4(state, h);
    const float u = to_float(static_cast<const T *>(a.u)[n * a.u_stride + k]);
    const float raw = to_float(static_cast<const T *>(a.dt)[n * a.dt_stride + k]) + (a.dt_bias ? a.dt_bias[k] : 0.f);
    const float dt = a.softplus ? softplus(raw) : raw;
    const T *b = static_cast<const T *>(a.b) + n * a.b_stride + group * N + lane * 4;
    const T *c = static_cast<const T *>(a.c) + n * a.c_stride + group * N + lane * 4;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = fmaf(exp2_approx(dt * (A[i] * kLog2e)), h[i], dt * u * to_float(b[i]));
        sum = fmaf(to_float(c[i]), h[i], sum);
    }
#pragma unroll
    for (int o = P / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!live) return;
    *reinterpret_cast<float4 *>(state) = make_float4(h[0], h[1], h[2], h[3]);
    if (lane == 0) {
        if (a.d) sum = fmaf(a.d[k], u, sum);
        if (a.z) sum *= silu(to_float(static_cast<const T *>(a.z)[n * a.z_stride + k]));
        y[d] = from_float<T>(sum);
    }
}

template <class T, int N>
cudaError_t launch_scan_as(const sq_scan_args &a, bool step, cudaStream_t s) {
    constexpr int CH = kScanThreads / (N / kPerLane);
    if (step) {
        const unsigned grid = unsigned((a.channels + CH - 1) / CH);
        scan_step_kernel<T, N><<<dim3(unsigned(a.num_seqs), grid), kScanThreads, 0, s>>>(a);
    } else {
        const int per = a.channels / a.groups;
        const unsigned grid = unsigned(a.groups * ((per + CH - 1) / CH));
        scan_kernel<T, N><<<dim3(unsigned(a.num_seqs), grid), kScanThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_scan(const sq_scan_args &a, bool step, cudaStream_t s) {
    switch (a.states) {
        case 4: return launch_scan_as<T, 4>(a, step, s);
        case 8: return launch_scan_as<T, 8>(a, step, s);
        case 16: return launch_scan_as<T, 16>(a, step, s);
        case 32: return launch_scan_as<T, 32>(a, step, s);
        default: return launch_scan_as<T, 64>(a, step, s);
    }
}

int32_t scan_entry(const sq_scan_args *args, bool step, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_scan_args &a = *args;
    if (a.tokens < 0 || a.num_seqs < 0 || a.channels < 1 || a.groups < 1 || (a.slots && a.num_slots < 1)) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16) return SQ_ERR_ARGUMENT;
    if (a.channels % a.groups || a.u_stride < 0 || a.dt_stride < 0 || a.z_stride < 0 || a.b_stride < 0 || a.c_stride < 0)
        return SQ_ERR_SHAPE;
    if (a.states != 4 && a.states != 8 && a.states != 16 && a.states != 32 && a.states != 64) return SQ_ERR_UNSUPPORTED;
    if (a.channels > (1 << 18)) return SQ_ERR_UNSUPPORTED;
    if (a.num_seqs == 0) return SQ_OK;
    if (!a.a || (a.tokens > 0 && (!a.u || !a.dt || !a.b || !a.c || !a.y))) return SQ_ERR_ARGUMENT;
    if (step ? !a.final_state : !a.cu_seqlens) return SQ_ERR_ARGUMENT;
    if (!aligned16(a.a) || !aligned16(a.initial_state) || !aligned16(a.final_state)) return SQ_ERR_SHAPE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? launch_scan<float>(a, step, s)
                          : a.dtype == SQ_BF16 ? launch_scan<__nv_bfloat16>(a, step, s)
                                               : launch_scan<__half>(a, step, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_selective_scan(const sq_scan_args *args, sq_stream_t stream) { return sq::scan_entry(args, false, stream); }

extern "C" int32_t sq_selective_scan_step(const sq_scan_args *args, sq_stream_t stream) {
    return sq::scan_entry(args, true, stream);
}

extern "C" int64_t sq_selective_scan_workspace_bytes(int32_t tokens, int32_t num_seqs, int32_t channels, int32_t states, int32_t groups) {
    if (tokens < 0 || num_seqs < 0 || channels < 1 || states < 1 || groups < 1) return -1;
    return 0;
}
