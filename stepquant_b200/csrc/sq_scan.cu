// Selective state space scan, for prompts (concatenated sequences) and for
// single tokens.  Channel d of group G = d / (channels / groups), state n:
//
//   dt' = softplus(dt + dt_bias)
//   h[d, n] <- exp(dt' A[d, n]) h[d, n] + dt' u B[G, n]
//   y[d] = (sum_n C[G, n] h[d, n] + D[d] u) silu(z)
//
// h, A and every intermediate are fp32; y is rounded once to the input's type.
//
// Prompts (scan_kernel): four states a lane, N / 4 lanes a channel; a CTA of 128
// lanes walks its channels through the tokens in tiles of 32.  Per tile the CTA
// forms dt' and dt' u once per (token, channel) in shared memory (two special
// functions, against N exponentials), the lanes run the recurrence in registers,
// four tokens at a time so that the loads and exponentials of a group do not wait
// on its chain h, and the outputs leave through shared memory.  The next tile's
// inputs are loaded before the recurrence of this one.
// Bound by the special function unit: one exponential per (token, channel,
// state) at 16 a clock and SM.
//
// Few channels and sequences: the tokens are cut into chunks.  A first pass gives
// each chunk's state from zero and its sum of dt' (the decay of a chunk is
// exp(A sum dt')), a second joins them along each sequence, the third is the scan
// of every chunk from its state.  Twice the exponentials, on many more lanes.
#include "sq_rows.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kScanThreads = 128;
constexpr int kTile = 32;     // tokens of a tile
constexpr int kPerLane = 4;   // states of a lane
constexpr int kUnroll = 4;    // tokens of a group
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// expf, not its fast form: far below zero softplus is the exponential, and the
// step size scales every input of the state.
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

// A lane's four entries of a state or A row (16-byte aligned: N is a multiple of 4).
__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// Four channels of a token: one load of 8 or 16 bytes, or (rows not aligned for
// it, or the last channels of a group) the first n singly.
template <class T>
struct Quad {
    alignas(4 * sizeof(T)) T v[4];
    __device__ __forceinline__ void load(const T *p, bool whole, int n) {
        if (whole) {
            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
            else *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void store(T *p, bool whole, int n) const {
        if (whole) {
            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(v);
            else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) p[i] = v[i];
        }
    }
};

// Workspace of the chunked scan: a state per (chunk, channel), then a sum of dt'.
struct Chunks {
    int length;     // tokens of a chunk; 0: whole sequences
    float *state;
    float *step_sum;
};

enum ScanPass { kWhole, kChunkState, kChunkScan };

template <class T, int N, int PASS>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(sq_scan_args a, Chunks chunks, bool vec) {
    constexpr int P = N / kPerLane;              // lanes of a channel
    constexpr int CH = kScanThreads / P;         // channels of the CTA
    constexpr int TILE = P > 1 ? kTile : kTile / 2;  // tokens of a tile (a lane a channel: shared memory for half)
    constexpr int QUADS = CH / 4, ROWS = kScanThreads / QUADS;  // a thread's quad of channels, rows of a load
    constexpr int EACH = TILE / ROWS > 0 ? TILE / ROWS : 1;
    __shared__ float2 step[TILE][CH];           // dt', dt' u
    __shared__ float ys[PASS == kChunkState ? 1 : TILE][PASS == kChunkState ? 1 : CH];
    __shared__ float4 bs[TILE][P], cs[TILE][P];
    const int tid = threadIdx.x, lane = tid % P, ch = tid / P;
    const int per = a.channels / a.groups, tiles = (per + CH - 1) / CH;  // CTAs of a group
    const int group = blockIdx.y / tiles, first = (blockIdx.y - group * tiles) * CH;
    const int live = min(CH, per - first), d0 = group * per + first;

    // ---- the tokens of this CTA
    const int n = PASS == kWhole ? blockIdx.x : sequence_of(a.cu_seqlens, a.num_seqs, a.tokens, chunks.length, blockIdx.x);
    const int2 seq = sequence_range(a.cu_seqlens, n, a.tokens);
    int begin = seq.x, end = seq.y;
    bool many = false;  // the sequence has several chunks
    if (PASS != kWhole) {
        const int64_t part = blockIdx.x - (seq.x / chunks.length + int64_t(n));
        if (part < 0 || (part > 0 && part * chunks.length >= seq.y - seq.x)) return;
        many = seq.y - seq.x > chunks.length;
        begin = seq.x + int(part) * chunks.length;
        end = min(seq.y, begin + chunks.length);
        if (PASS == kChunkState && end == seq.y) return;  // no chunk follows
    }
    T *y = static_cast<T *>(a.y) + d0;
    const int64_t row = state_row(a.slots, n, a.num_slots, PASS == kChunkState ? nullptr : a.status);
    if (row < 0) {
        if (PASS != kChunkState)
            for (int64_t i = tid; i < (end - begin) * int64_t(CH); i += kScanThreads)
                if (i % CH < live) y[(begin + i / CH) * a.channels + i % CH] = from_float<T>(0.f);
        return;
    }

    // ---- this lane's states
    const int mine = min(ch, live - 1);  // lanes past the group's channels follow its last
    float A[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    load4(a.a + int64_t(d0 + mine) * N + lane * 4, A);
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] *= kLog2e;
    const int64_t at = (row * a.channels + d0 + mine) * N + lane * 4;
    const int64_t kept = (int64_t(blockIdx.x) * a.channels + d0 + mine) * N + lane * 4;
    if (PASS == kChunkScan && many) load4(chunks.state + kept, h);
    else if (PASS != kChunkState && a.initial_state) load4(a.initial_state + at, h);
    float total = 0.f;  // sum of dt' (first lane of the channel)

    // ---- this thread's share of a tile's loads: rows r, r + ROWS, ... of one quad of channels
    const int quad = tid % QUADS * 4, row0 = tid / QUADS, width = max(0, min(4, live - quad));
    const bool whole = vec && width == 4;
    const T *u = static_cast<const T *>(a.u) + d0 + quad, *dt = static_cast<const T *>(a.dt) + d0 + quad;
    const T *z = a.z ? static_cast<const T *>(a.z) + d0 + quad : nullptr;
    const T *b = static_cast<const T *>(a.b) + group * N, *c = static_cast<const T *>(a.c) + group * N;
    constexpr int BC = (TILE * N + kScanThreads - 1) / kScanThreads;  // entries of B (and C) a thread loads a tile
    float bias[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = a.dt_bias && i < width ? a.dt_bias[d0 + quad + i] : 0.f;
        skip[i] = PASS != kChunkState && a.d && i < width ? a.d[d0 + quad + i] : 0.f;
    }
    Quad<T> next_dt[EACH], next_u[EACH], next_z[EACH];
    T next_b[BC], next_c[BC];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int64_t t = t0 + row0 + e * ROWS;
            if (row0 + e * ROWS < TILE && t < end) {
                next_dt[e].load(dt + t * a.dt_stride, whole, width);
                next_u[e].load(u + t * a.u_stride, whole, width);
                if (PASS != kChunkState && z) next_z[e].load(z + t * a.z_stride, whole, width);
            }
        }
#pragma unroll
        for (int e = 0; e < BC; ++e) {
            const int i = e * kScanThreads + tid;
            const int64_t t = t0 + i / N;
            if (i >= TILE * N) continue;
            next_b[e] = t < end ? b[t * a.b_stride + i % N] : from_float<T>(0.f);
            if (PASS != kChunkState) next_c[e] = t < end ? c[t * a.c_stride + i % N] : from_float<T>(0.f);
        }
    };
    // dt', dt' u, B and C of the fetched tile into shared memory; rows past the end leave the state alone.
    auto put = [&](int t0) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int r = row0 + e * ROWS;
            if (r >= TILE) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = to_float(next_dt[e].v[i]) + bias[i];
                const float s = t0 + r < end ? (a.softplus ? softplus(x) : x) : 0.f;
                step[r][quad + i] = make_float2(s, t0 + r < end ? s * to_float(next_u[e].v[i]) : 0.f);
            }
        }
#pragma unroll
        for (int e = 0; e < BC; ++e) {
            const int i = e * kScanThreads + tid;
            if (i >= TILE * N) continue;
            reinterpret_cast<float *>(bs)[i] = to_float(next_b[e]);
            if (PASS != kChunkState) reinterpret_cast<float *>(cs)[i] = to_float(next_c[e]);
        }
    };

    if (begin < end) {
        fetch(begin);
        put(begin);
    }
    __syncthreads();
    for (int t0 = begin; t0 < end; t0 += TILE) {
        Quad<T> now_u[EACH], now_z[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) now_u[e] = next_u[e], now_z[e] = next_z[e];
        if (t0 + TILE < end) fetch(t0 + TILE);
        const int count = min(TILE, end - t0);
        for (int t = 0; t < count; t += kUnroll) {  // rows past the end have dt' = 0
            float2 s[kUnroll];
            float4 bv[kUnroll], cv[kUnroll];
            float decay[kUnroll][4], sum[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                s[j] = step[t + j][ch];
                bv[j] = bs[t + j][lane];
                if (PASS != kChunkState) cv[j] = cs[t + j][lane];
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) decay[j][i] = exp2_approx(s[j].x * A[i]);
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const float bb[4] = {bv[j].x, bv[j].y, bv[j].z, bv[j].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = fmaf(decay[j][i], h[i], s[j].y * bb[i]);
                if (PASS == kChunkState) {
                    total += s[j].x;
                } else {
                    const float cc[4] = {cv[j].x, cv[j].y, cv[j].z, cv[j].w};
                    sum[j] = fmaf(cc[3], h[3], fmaf(cc[2], h[2], fmaf(cc[1], h[1], cc[0] * h[0])));
                }
            }
            if (PASS != kChunkState) {
#pragma unroll
                for (int o = P / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int j = 0; j < kUnroll; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
                if (lane == 0) {
#pragma unroll
                    for (int j = 0; j < kUnroll; ++j) ys[t + j][ch] = sum[j];
                }
            }
        }
        __syncthreads();
        if (PASS != kChunkState) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int r = row0 + e * ROWS;
                if (r >= count || width == 0) continue;
                Quad<T> out;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = ys[r][quad + i];
                    if (a.d) v = fmaf(skip[i], to_float(now_u[e].v[i]), v);
                    if (z) v *= silu(to_float(now_z[e].v[i]));
                    out.v[i] = from_float<T>(v);
                }
                out.store(y + quad + int64_t(t0 + r) * a.channels, whole, width);
            }
        }
        if (t0 + TILE < end) put(t0 + TILE);
        __syncthreads();
    }
    if (ch >= live) return;
    if (PASS == kChunkState) {
        *reinterpret_cast<float4 *>(chunks.state + kept) = make_float4(h[0], h[1], h[2], h[3]);
        if (lane == 0) chunks.step_sum[int64_t(blockIdx.x) * a.channels + d0 + ch] = total;
    } else if (a.final_state && end == seq.y) {
        *reinterpret_cast<float4 *>(a.final_state + at) = make_float4(h[0], h[1], h[2], h[3]);
    }
}

// Along each sequence of several chunks: the state that every chunk starts from.
__global__ void join_kernel(sq_scan_args a, Chunks chunks) {
    const int64_t i = int64_t(blockIdx.y) * blockDim.x + threadIdx.x;  // (channel, state)
    const int n = blockIdx.x;
    if (i >= int64_t(a.channels) * a.states) return;
    const int2 seq = sequence_range(a.cu_seqlens, n, a.tokens);
    const int count = (seq.y - seq.x + chunks.length - 1) / chunks.length;
    if (count < 2) return;
    const int64_t row = state_row(a.slots, n, a.num_slots, nullptr);
    if (row < 0) return;
    const int64_t size = int64_t(a.channels) * a.states, d = i / a.states;
    const float A = a.a[i] * kLog2e;
    float h = a.initial_state ? a.initial_state[row * size + i] : 0.f;
    const int64_t base = seq.x / chunks.length + int64_t(n);
    for (int k = 0; k < count; ++k) {
        float *at = chunks.state + (base + k) * size + i;
        const float own = k + 1 < count ? *at : 0.f, sum = k + 1 < count ? chunks.step_sum[(base + k) * a.channels + d] : 0.f;
        *at = h;
        h = fmaf(exp2_approx(A * sum), h, own);
    }
}

// One token of each request: N / 4 lanes a channel, the state read and written
// once.  A lane takes R requests, their states in flight together; of the R
// steps and gates of its channel each lane forms its share.
template <class T, int N, int R>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(sq_scan_args a) {
    constexpr int P = N / kPerLane;
    constexpr int SHARE = R > P ? R / P : 1;  // requests whose scalars a lane forms
    const int lane = threadIdx.x % P, n0 = blockIdx.x * R;
    const int d = (blockIdx.y * kScanThreads + threadIdx.x) / P;
    const bool live = d < a.channels;
    const int k = live ? d : a.channels - 1, group = k / (a.channels / a.groups);
    int64_t rows[R];
    float h[R][4], A[4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        rows[r] = n0 + r < a.num_seqs ? state_row(a.slots, n0 + r, a.num_slots, a.status) : -1;
        if (rows[r] >= 0) load4(a.final_state + (rows[r] * a.channels + k) * N + lane * 4, h[r]);
    }
    load4(a.a + int64_t(k) * N + lane * 4, A);
    float dt_mine[SHARE], u_mine[SHARE], z_mine[SHARE];
    const float bias = a.dt_bias ? a.dt_bias[k] : 0.f, skip = a.d ? a.d[k] : 0.f;
#pragma unroll
    for (int q = 0; q < SHARE; ++q) {
        const int r = lane + q * P;
        const int64_t n = n0 + r;
        dt_mine[q] = u_mine[q] = z_mine[q] = 0.f;
        if (r < R && n < a.num_seqs) {
            u_mine[q] = to_float(static_cast<const T *>(a.u)[n * a.u_stride + k]);
            const float raw = to_float(static_cast<const T *>(a.dt)[n * a.dt_stride + k]) + bias;
            if (a.z) z_mine[q] = to_float(static_cast<const T *>(a.z)[n * a.z_stride + k]);
            dt_mine[q] = a.softplus ? softplus(raw) : raw;
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int from = (threadIdx.x & 31) / P * P + r % P;
        const float dt = __shfl_sync(0xffffffffu, dt_mine[r / P % SHARE], from), u = __shfl_sync(0xffffffffu, u_mine[r / P % SHARE], from);
        const int64_t n = n0 + r;
        float sum = 0.f;
        if (rows[r] >= 0) {
            const T *b = static_cast<const T *>(a.b) + n * a.b_stride + group * N + lane * 4;
            const T *c = static_cast<const T *>(a.c) + n * a.c_stride + group * N + lane * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[r][i] = fmaf(exp2_approx(dt * (A[i] * kLog2e)), h[r][i], dt * u * to_float(b[i]));
                sum = fmaf(to_float(c[i]), h[r][i], sum);
            }
            if (live)
                *reinterpret_cast<float4 *>(a.final_state + (rows[r] * a.channels + k) * N + lane * 4) =
                    make_float4(h[r][0], h[r][1], h[r][2], h[r][3]);
        }
#pragma unroll
        for (int o = P / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (live && lane == r % P && n < a.num_seqs) {
            if (a.d) sum = fmaf(skip, u, sum);
            if (a.z) sum *= silu(z_mine[r / P % SHARE]);
            static_cast<T *>(a.y)[n * a.channels + d] = from_float<T>(rows[r] >= 0 ? sum : 0.f);
        }
    }
}

// Tokens of a chunk, 0 for whole sequences: cut where the lanes of whole
// sequences leave most of the 592 warp schedulers without a warp.
int chunk_length(int tokens, int seqs, int channels, int states) {
    const int64_t warps = int64_t(channels) * (states / kPerLane) / 32 + 1;
    if (seqs * warps >= 592 * 3 || tokens < 256) return 0;
    const int64_t wanted = 592 * 6 / warps;  // chunks that fill them
    int64_t length = (tokens / (wanted > 1 ? wanted : 1) + kTile - 1) / kTile * kTile;
    if (length < 64) length = 64;
    return length * 2 > tokens / seqs * int64_t(3) ? 0 : int(length);
}

template <class T, int N>
cudaError_t launch_scan_as(const sq_scan_args &a, bool step, cudaStream_t s) {
    constexpr int CH = kScanThreads / (N / kPerLane);
    if (step) {
        const unsigned grid = unsigned((a.channels + CH - 1) / CH);
        if (int64_t(a.num_seqs) * grid < 148 * 16) scan_step_kernel<T, N, 1><<<dim3(unsigned(a.num_seqs), grid), kScanThreads, 0, s>>>(a);
        else scan_step_kernel<T, N, 4><<<dim3(unsigned((a.num_seqs + 3) / 4), grid), kScanThreads, 0, s>>>(a);
        return cudaGetLastError();
    }
    const int per = a.channels / a.groups;
    const unsigned columns = unsigned(a.groups * ((per + CH - 1) / CH));
    const int64_t size = sizeof(T);
    auto quads = [&](const void *p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0; };
    const bool vec = per % 4 == 0 && quads(a.u, a.u_stride) && quads(a.dt, a.dt_stride) && (!a.z || quads(a.z, a.z_stride)) &&
                     quads(a.y, a.channels);
    Chunks chunks{};
    if (a.workspace) chunks.length = chunk_length(a.tokens, a.num_seqs, a.channels, a.states);
    if (!chunks.length) {
        scan_kernel<T, N, kWhole><<<dim3(unsigned(a.num_seqs), columns), kScanThreads, 0, s>>>(a, chunks, vec);
        return cudaGetLastError();
    }
    const int64_t count = a.tokens / chunks.length + a.num_seqs;
    chunks.state = static_cast<float *>(a.workspace);
    chunks.step_sum = chunks.state + count * a.channels * N;
    const dim3 grid(unsigned(count), columns);
    scan_kernel<T, N, kChunkState><<<grid, kScanThreads, 0, s>>>(a, chunks, vec);
    join_kernel<<<dim3(unsigned(a.num_seqs), unsigned((int64_t(a.channels) * N + 255) / 256)), 256, 0, s>>>(a, chunks);
    scan_kernel<T, N, kChunkScan><<<grid, kScanThreads, 0, s>>>(a, chunks, vec);
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
    if (a.channels > (1 << 18) || a.groups > (1 << 14)) return SQ_ERR_UNSUPPORTED;
    if (a.num_seqs == 0) return SQ_OK;
    if (!a.a || (a.tokens > 0 && (!a.u || !a.dt || !a.b || !a.c || !a.y))) return SQ_ERR_ARGUMENT;
    if (step ? !a.final_state : !a.cu_seqlens) return SQ_ERR_ARGUMENT;
    if (!aligned16(a.a) || !aligned16(a.initial_state) || !aligned16(a.final_state) || !aligned16(a.workspace)) return SQ_ERR_SHAPE;
    if (!step && a.workspace &&
        a.workspace_bytes < sq_selective_scan_workspace_bytes(a.tokens, a.num_seqs, a.channels, a.states, a.groups))
        return SQ_ERR_CAPACITY;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? launch_scan<float>(a, step, s)
                          : a.dtype == SQ_BF16 ? launch_scan<__nv_bfloat16>(a, step, s)
                                               : launch_scan<__half>(a, step, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

}  // namespace
}  // namespace sq

extern "C" int64_t sq_selective_scan_workspace_bytes(int32_t tokens, int32_t num_seqs, int32_t channels, int32_t states,
                                                     int32_t groups) {
    if (tokens < 0 || num_seqs < 0 || channels < 1 || states < 1 || groups < 1) return -1;
    const int length = num_seqs ? sq::chunk_length(tokens, num_seqs, channels, states) : 0;
    if (!length) return 0;
    return (int64_t(tokens / length) + num_seqs) * channels * (states + 1) * int64_t(sizeof(float));
}

extern "C" int32_t sq_selective_scan(const sq_scan_args *args, sq_stream_t stream) { return sq::scan_entry(args, false, stream); }

extern "C" int32_t sq_selective_scan_step(const sq_scan_args *args, sq_stream_t stream) {
    return sq::scan_entry(args, true, stream);
}
