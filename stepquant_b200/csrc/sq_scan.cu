// Selective state space scan, for prompts (concatenated sequences) and for
// single tokens.  Channel d of group G = d / (channels / groups), state n:
//
//   dt' = softplus(dt + dt_bias)
//   h[d, n] <- exp(dt' A[d, n]) h[d, n] + dt' u B[G, n]
//   y[d] = (sum_n C[G, n] h[d, n] + D[d] u) silu(z)
//
// h, A and every intermediate are fp32; y is rounded once to the input's type.
//
// Prompts (scan_kernel): a lane holds up to 16 states of one channel and walks it
// through the tokens, so dt', the gate and the sum over N are formed where they
// are used and only more than 16 states need an exchange.  B and C, the same for
// all channels of a group, are read from shared memory by broadcast.  A CTA of 128
// lanes takes its tokens in tiles; the raw rows of the next tile are in flight
// (cp.async of the 16-byte pieces that cover a row, so rows of any alignment take
// one path) while a tile is worked on.  Four tokens at a time, so that the
// exponentials and gates of one do not wait on the chain h of the others.
// Bound by the special function unit (one exponential per token, channel and
// state at 16 a clock and SM, four more per token and channel) and, next to it, by
// issue: 145 instructions for 20 special functions of a warp and token.  Measured
// at 8192 tokens x 4096 channels x 16 states in 32 prompts 200 us, 0.72 of that
// unit's rate.  Four states a lane with the sums exchanged between lanes took 301
// us (221 instructions for the same states), softplus and gate behind a run-time
// branch 230 us: the compiler mixes the tokens of a group only without one.
//
// Few channels and sequences: the tokens are cut into chunks.  A first pass gives
// each chunk's state from zero and its sum of dt' (the decay of a chunk is
// exp(A sum dt')), a second joins them along each sequence, the third is the scan
// of every chunk from its state.  Twice the exponentials, on many more lanes: one
// prompt of 8192 tokens x 2048 channels 85 + 13 + 104 us, against 1430 us whole.
#include <type_traits>
#include "sq_rows.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kScanThreads = 128;
constexpr int kPerLane = 4;   // states of a lane of the single-token kernel
constexpr int kGroup = 4;     // tokens of a prompt worked on together
constexpr unsigned kGridRows = 32768;  // groups of requests along a grid's second axis, the rest along its third
constexpr float kLog2eRest = 1.92596299e-8f;  // log2(e) - kLog2e

// log(1 + e^x), x = raw + bias, as max(x, 0) + log1p(e^-|x|), off by less than 16 * 2^-24 of
// itself (4 measured; zero below 2^-126): the step size scales every input of the state, and far
// below zero softplus is the exponential alone.  So the rounding errors of the sum (two-sum: the
// larger of the two may be either) and of its product with log2(e) are carried into the
// exponential to first order; log1p(e) = 2 atanh(e / (2 + e)) is its series to the 13th power
// (the argument is at most 1/3).  NaN stays NaN, an infinite x gives 0 or itself.
__device__ __forceinline__ float softplus(float raw, float bias) {
    const float x = raw + bias, part = x - raw;
    const float lost = fminf((raw - (x - part)) + (bias - part), 1.f);  // of x; NaN where x is infinite
    const float m = fminf(fabsf(x), 128.f), y = m * kLog2e;
    const float rest = fmaf(m, kLog2eRest, fmaf(m, kLog2e, -y));
    const float off = fmaf(rest, 0.6931471806f, __uint_as_float(__float_as_uint(lost) ^ (__float_as_uint(x) & 0x80000000u)));  // of |x|
    const float p = exp2_approx(-y), e = fmaf(-p, off, p);
    const float q = e * reciprocal_approx(2.f + e), q2 = q * q;
    float s = fmaf(q2, 1.f / 13.f, 1.f / 11.f);
    s = fmaf(q2, s, 1.f / 9.f);
    s = fmaf(q2, s, 1.f / 7.f);
    s = fmaf(q2, s, 1.f / 5.f);
    s = fmaf(q2, s, 1.f / 3.f);
    s = fmaf(q2 * s, q, q);
    float top;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(top) : "f"(x));
    return fmaf(2.f, s, top);
}

// A lane's four entries of a state or A row (16-byte aligned: N is a multiple of 4).
__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// The 16-byte pieces that cover `bytes` bytes from p on, piece `i` into a row of
// shared memory; nothing past the last byte is read (a piece may begin before p:
// in the row before, or in the padding below a tensor's first row).
__device__ __forceinline__ void cover(unsigned char *row, const void *p, int bytes, int i) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p), piece = (from & ~uintptr_t(15)) + 16 * i;
    const int64_t left = int64_t(from) + bytes - int64_t(piece);
    if (left <= 0) return;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(row + 16 * i))),
                 "l"(piece), "r"(int(left < 16 ? left : 16)) : "memory");
}
// Workspace of the chunked scan: a state per (chunk, channel), then a sum of dt'.
struct Chunks {
    int length;     // tokens of a chunk; 0: whole sequences
    float *state;
    float *step_sum;
};

enum ScanPass { kWhole, kChunkState, kChunkScan };

// Sizes of a CTA and its shared memory.
template <class T, int N>
struct ScanShape {
    static constexpr int SN = N < 16 ? N : 16;     // states of a lane
    static constexpr int P = N / SN;               // lanes of a channel
    static constexpr int CH = kScanThreads / P;    // channels of the CTA
    static constexpr int TILE = 16;           // tokens of a tile
    // Raw rows with their cover, whole 16-byte pieces (4 states of 16 bits are half a piece).
    static constexpr int kRow = CH * sizeof(T) + 16, kBcRow = (N * sizeof(T) + 15) / 16 * 16 + 16;
    static_assert(kRow % 16 == 0 && kBcRow % 16 == 0, "cp.async writes 16-byte aligned pieces");
    static constexpr int kStage = TILE * (3 * kRow + 2 * kBcRow);                  // dt, u, z, B, C
    static constexpr int kBc = TILE * N * 4;
    static constexpr int kBytes = 2 * kBc + 2 * kStage;
};

// USUAL: softplus and (where there are outputs) a gate, known to the compiler so that the
// tokens of a group have no branches between them; else as the arguments say.  Whole
// sequences: the CTAs past `parts` clear the tokens of no sequence.
template <class T, int N, int PASS, bool USUAL>
__global__ void __launch_bounds__(kScanThreads, 4) scan_kernel(sq_scan_args a, Chunks chunks, unsigned parts) {
    using S = ScanShape<T, N>;
    constexpr int SN = S::SN, P = S::P, CH = S::CH, TILE = S::TILE;
    constexpr bool OUT = PASS != kChunkState;
    extern __shared__ __align__(16) unsigned char smem[];
    float4 *bs = reinterpret_cast<float4 *>(smem), *cs = reinterpret_cast<float4 *>(smem + S::kBc);  // [TILE][N]
    unsigned char *raw = smem + 2 * S::kBc;
    const int tid = threadIdx.x, lane = tid % P, ch = tid / P;
    const int per = a.channels / a.groups, tiles = (per + CH - 1) / CH;  // CTAs of a group
    const int group = blockIdx.y / tiles, first = (blockIdx.y - group * tiles) * CH;
    const int live = min(CH, per - first), d0 = group * per + first;
    if (PASS == kWhole && blockIdx.x >= parts) {
        clear_outside(a.y, int64_t(a.channels) * sizeof(T), a.cu_seqlens, a.num_seqs, a.tokens,
                      (blockIdx.x - parts) * gridDim.y + blockIdx.y, (gridDim.x - parts) * gridDim.y);
        return;
    }
    T *y = static_cast<T *>(a.y) + d0;

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
        end = int(min(int64_t(seq.y), int64_t(begin) + chunks.length));
        if (PASS == kChunkState && end == seq.y) return;  // no chunk follows
    }
    const int64_t row = state_row(a.slots, n, a.num_slots, OUT ? a.status : nullptr);
    if (row < 0) {
        if (OUT)
            for (int64_t i = tid; i < (end - begin) * int64_t(CH); i += kScanThreads)
                if (i % CH < live) y[(begin + i / CH) * a.channels + i % CH] = from_float<T>(0.f);
        return;
    }

    // ---- raw rows of a tile: a power of two of threads a row, its pieces among them
    const T *u = static_cast<const T *>(a.u) + d0, *dt = static_cast<const T *>(a.dt) + d0;
    const T *z = a.z ? static_cast<const T *>(a.z) + d0 : nullptr;
    const T *b = static_cast<const T *>(a.b) + group * N, *c = static_cast<const T *>(a.c) + group * N;
    constexpr int kU = TILE * S::kRow, kZ = 2 * kU, kB = 3 * kU, kC = kB + TILE * S::kBcRow;  // offsets in a stage (dt at 0)
    constexpr int PIECES = S::kRow / 16, LANES = PIECES <= 5 ? 4 : PIECES <= 9 ? 8 : PIECES <= 17 ? 16 : 32;
    constexpr int BC_PIECES = S::kBcRow / 16, BC_LANES = BC_PIECES <= 4 ? 4 : BC_PIECES <= 8 ? 8 : BC_PIECES <= 16 ? 16 : 32;
    constexpr int PASS_ROWS = kScanThreads / LANES, BC_ROWS = kScanThreads / BC_LANES;
    const int bytes = live * int(sizeof(T)), bc_bytes = N * int(sizeof(T));
    const T *fetch_dt = dt + (int64_t(begin) + tid / LANES) * a.dt_stride, *fetch_u = u + (int64_t(begin) + tid / LANES) * a.u_stride;
    const T *fetch_z = OUT && z ? z + (int64_t(begin) + tid / LANES) * a.z_stride : nullptr;
    const T *fetch_b = b + (int64_t(begin) + tid / BC_LANES) * a.b_stride, *fetch_c = c + (int64_t(begin) + tid / BC_LANES) * a.c_stride;
    auto fetch = [&](int t0, int stage) {  // the tile after the one fetched before
        const int count = min(TILE, end - t0);
        unsigned char *to = raw + stage * S::kStage + tid / LANES * S::kRow;
#pragma unroll
        for (int r = 0; r < TILE; r += PASS_ROWS) {
            if (r + tid / LANES < count) {
#pragma unroll
                for (int p = 0; p < PIECES; p += LANES)  // a cover is one piece longer than its row
                    if (p == 0 || tid % LANES == 0) {
                        cover(to + r * S::kRow, fetch_dt, bytes, tid % LANES + p);
                        cover(to + kU + r * S::kRow, fetch_u, bytes, tid % LANES + p);
                        if (OUT && (USUAL || z)) cover(to + kZ + r * S::kRow, fetch_z, bytes, tid % LANES + p);
                    }
            }
            constexpr int DONE = PASS_ROWS < TILE ? PASS_ROWS : TILE;
            fetch_dt += DONE * a.dt_stride;
            fetch_u += DONE * a.u_stride;
            if (OUT && (USUAL || z)) fetch_z += DONE * a.z_stride;
        }
        to = raw + stage * S::kStage + tid / BC_LANES * S::kBcRow;
#pragma unroll
        for (int r = 0; r < TILE; r += BC_ROWS) {
            if (r + tid / BC_LANES < count && tid % BC_LANES < BC_PIECES) {
                cover(to + kB + r * S::kBcRow, fetch_b, bc_bytes, tid % BC_LANES);
                if (OUT) cover(to + kC + r * S::kBcRow, fetch_c, bc_bytes, tid % BC_LANES);
            }
            constexpr int DONE = BC_ROWS < TILE ? BC_ROWS : TILE;
            fetch_b += DONE * a.b_stride;
            if (OUT) fetch_c += DONE * a.c_stride;
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;\n" ::: "memory"); };
    if (begin < end) fetch(begin, 0);
    commit();

    // ---- this lane's states, in pairs
    const int k = min(ch, live - 1), d = d0 + k;  // lanes past the group's channels follow its last
    const int64_t at = (row * a.channels + d) * N + lane * SN, kept = (int64_t(blockIdx.x) * a.channels + d) * N + lane * SN;
    float2 A[SN / 2], h[SN / 2];
#pragma unroll
    for (int i = 0; i < SN / 4; ++i) {
        float v[4];
        load4(a.a + int64_t(d) * N + lane * SN + 4 * i, v);
        A[2 * i] = make_float2(v[0] * kLog2e, v[1] * kLog2e), A[2 * i + 1] = make_float2(v[2] * kLog2e, v[3] * kLog2e);
        v[0] = v[1] = v[2] = v[3] = 0.f;
        if (PASS == kChunkScan && many) load4(chunks.state + kept + 4 * i, v);
        else if (OUT && a.initial_state) load4(a.initial_state + at + 4 * i, v);
        h[2 * i] = make_float2(v[0], v[1]), h[2 * i + 1] = make_float2(v[2], v[3]);
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f;
    const float skip = OUT && a.d ? a.d[d] : 0.f;
    float total = 0.f;  // sum of dt'

    int stage = 0;
    y += int64_t(begin) * a.channels + ch;
    const bool stores = ch < live && lane == 0;
    // Byte offsets of this lane's value in the raw rows: the alignment of row t within 16 bytes, plus the channel.
    const uint32_t dt_low = uint32_t(reinterpret_cast<uintptr_t>(dt)), dt_step = uint32_t(a.dt_stride * sizeof(T));
    const uint32_t u_low = uint32_t(reinterpret_cast<uintptr_t>(u)), u_step = uint32_t(a.u_stride * sizeof(T));
    const uint32_t z_low = uint32_t(reinterpret_cast<uintptr_t>(z)), z_step = uint32_t(a.z_stride * sizeof(T));
    const uint32_t b_low = uint32_t(reinterpret_cast<uintptr_t>(b)), b_step = uint32_t(a.b_stride * sizeof(T));
    const uint32_t c_low = uint32_t(reinterpret_cast<uintptr_t>(c)), c_step = uint32_t(a.c_stride * sizeof(T));
    auto value = [&](const unsigned char *rows, int row_bytes, uint32_t low, uint32_t step, int t0, int r, int i) {
        return to_float(reinterpret_cast<const T *>(rows + r * row_bytes + ((low + uint32_t(t0 + r) * step) & 15))[i]);
    };
    for (int t0 = begin; t0 < end; t0 += TILE, stage ^= 1) {
        const unsigned char *from = raw + stage * S::kStage;
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        __syncthreads();  // this tile's rows have landed; the tile before is done with B and C
        const int count = min(TILE, end - t0);
        for (int i = tid; i < count * N; i += kScanThreads) {
            reinterpret_cast<float *>(bs)[i] = value(from + kB, S::kBcRow, b_low, b_step, t0, i / N, i % N);
            if (OUT) reinterpret_cast<float *>(cs)[i] = value(from + kC, S::kBcRow, c_low, c_step, t0, i / N, i % N);
        }
        __syncthreads();
        if (t0 + TILE < end) fetch(t0 + TILE, stage ^ 1);
        commit();
        auto tokens = [&](int t, auto group) {  // the next `group` tokens of the tile
            constexpr int U = decltype(group)::value;
            float s[U], in[U], un[U];
            float2 decay[U][SN / 2];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const float x = value(from, S::kRow, dt_low, dt_step, t0, t + j, k);
                un[j] = value(from + kU, S::kRow, u_low, u_step, t0, t + j, k);
                s[j] = USUAL || a.softplus ? softplus(x, bias) : x + bias;
                in[j] = s[j] * un[j];
                if (!OUT) total += s[j];
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int i = 0; i < SN / 2; ++i) {
                    const float2 x = mul2(make_float2(s[j], s[j]), A[i]);
                    decay[j][i] = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float2 sum = make_float2(0.f, 0.f);
                const float2 both = make_float2(in[j], in[j]);
#pragma unroll
                for (int i = 0; i < SN / 4; ++i) {
                    const float4 bv = bs[((t + j) * N + lane * SN) / 4 + i];
                    h[2 * i] = fma2(decay[j][2 * i], h[2 * i], mul2(both, make_float2(bv.x, bv.y)));
                    h[2 * i + 1] = fma2(decay[j][2 * i + 1], h[2 * i + 1], mul2(both, make_float2(bv.z, bv.w)));
                    if (OUT) {
                        const float4 cv = cs[((t + j) * N + lane * SN) / 4 + i];
                        sum = fma2(make_float2(cv.x, cv.y), h[2 * i], sum);
                        sum = fma2(make_float2(cv.z, cv.w), h[2 * i + 1], sum);
                    }
                }
                if (!OUT) continue;
                float v = sum.x + sum.y;
#pragma unroll
                for (int o = P / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                v = fmaf(skip, un[j], v);
                if (USUAL || z) v *= silu(value(from + kZ, S::kRow, z_low, z_step, t0, t + j, k));
                if (stores) *y = from_float<T>(v);
                y += a.channels;
            }
        };
        int t = 0;
        for (; t + kGroup <= count; t += kGroup) tokens(t, std::integral_constant<int, kGroup>());
        for (; t < count; ++t) tokens(t, std::integral_constant<int, 1>());
    }
    if (ch >= live) return;
#pragma unroll
    for (int i = 0; i < SN / 4; ++i) {
        const float4 v = make_float4(h[2 * i].x, h[2 * i].y, h[2 * i + 1].x, h[2 * i + 1].y);
        if (!OUT) *reinterpret_cast<float4 *>(chunks.state + kept + 4 * i) = v;
        else if (a.final_state && end == seq.y) *reinterpret_cast<float4 *>(a.final_state + at + 4 * i) = v;
    }
    if (!OUT && lane == 0) chunks.step_sum[int64_t(blockIdx.x) * a.channels + d] = total;
}

// Along each sequence of several chunks: the state that every chunk starts from.  The CTAs
// past the sequences clear the tokens of none.
__global__ void join_kernel(sq_scan_args a, Chunks chunks) {
    const int64_t i = int64_t(blockIdx.y) * blockDim.x + threadIdx.x;  // (channel, state)
    const int n = blockIdx.x;
    if (n == a.num_seqs) {
        clear_outside(a.y, int64_t(a.channels) * (a.dtype == SQ_F32 ? 4 : 2), a.cu_seqlens, a.num_seqs, a.tokens, blockIdx.y, gridDim.y);
        return;
    }
    if (i >= int64_t(a.channels) * a.states) return;
    const int2 seq = sequence_range(a.cu_seqlens, n, a.tokens);
    const int count = int((int64_t(seq.y) - seq.x + chunks.length - 1) / chunks.length);
    if (count < 2) return;
    const int64_t row = state_row(a.slots, n, a.num_slots, nullptr);
    if (row < 0) return;
    const int64_t size = int64_t(a.channels) * a.states, d = i / a.states;
    const float A = a.a[i] * kLog2e;
    float h = a.initial_state ? a.initial_state[row * size + i] : 0.f;
    const int64_t base = seq.x / chunks.length + int64_t(n);
    constexpr int B = 16;  // chunks whose loads are in flight together
    for (int k = 0; k < count; k += B) {
        float own[B], sum[B];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const bool in = k + j + 1 < count;  // of the last chunk nothing was kept
            own[j] = in ? chunks.state[(base + k + j) * size + i] : 0.f;
            sum[j] = in ? chunks.step_sum[(base + k + j) * a.channels + d] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (k + j < count) {
                chunks.state[(base + k + j) * size + i] = h;
                h = fmaf(exp2_approx(A * sum[j]), h, own[j]);
            }
    }
}

// Four values of a row, by one access where `whole`.
template <class T>
struct Quad {
    alignas(4 * sizeof(T)) T v[4];
    __device__ __forceinline__ void load(const T *p, bool whole) {
        if (whole) {
            if (sizeof(T) == 2) *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
            else *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p[i];
        }
    }
};

// One token of each request: N / 4 lanes a channel, the state read and written
// once.  A lane takes R requests, their states (and B and C) in flight together;
// of the R steps and gates of its channel each lane forms its share.  Bound by the
// states' bytes (8 a channel and state); `whole`: B and C rows are aligned for one
// access of four.  Measured at 4096 channels x 16 states: 512 requests in 57 us (5.0
// TB/s; one request a lane 95 us, eight 96 us), one request 2.7 us.
template <class T, int N, int R, bool USUAL>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(sq_scan_args a, bool whole) {
    constexpr int P = N / kPerLane;
    constexpr int SHARE = R > P ? R / P : 1;  // requests whose scalars a lane forms
    // Neighbouring CTAs take neighbouring channels: a request's state row is read through.
    const int lane = threadIdx.x % P, n0 = (blockIdx.z * kGridRows + blockIdx.y) * R;
    const int d = (blockIdx.x * kScanThreads + threadIdx.x) / P;
    const bool live = d < a.channels;
    const int k = live ? d : a.channels - 1, group = a.groups == 1 ? 0 : k / (a.channels / a.groups);
    // The requests' places, formed once a CTA: state (-1: none), u, dt, z, B, C, y.
    __shared__ int64_t place[7][R];
    if (threadIdx.x < R) {
        const int n = n0 + threadIdx.x;
        const int64_t row = n < a.num_seqs ? state_row(a.slots, n, a.num_slots, a.status) : -1;
        const int64_t in = min(n, a.num_seqs - 1);  // past the batch: read the last request's, write nothing
        place[0][threadIdx.x] = row < 0 ? -1 : row * a.channels * N;
        place[1][threadIdx.x] = in * a.u_stride;
        place[2][threadIdx.x] = in * a.dt_stride;
        place[3][threadIdx.x] = in * a.z_stride;
        place[4][threadIdx.x] = in * a.b_stride;
        place[5][threadIdx.x] = in * a.c_stride;
        place[6][threadIdx.x] = n < a.num_seqs ? int64_t(n) * a.channels : -1;
    }
    __syncthreads();
    int64_t rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = place[0][r];
    const int own = k * N + lane * 4, bc = group * N + lane * 4;  // below 2^24 and 2^20
    float A[4], h[R][4];
    Quad<T> b[R], c[R];
    T dt_raw[SHARE], u_raw[SHARE], z_raw[SHARE];
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (rows[r] >= 0) load4(a.final_state + rows[r] + own, h[r]);
#pragma unroll
    for (int q = 0; q < SHARE; ++q) {
        const int r = min(lane + q * P, R - 1);  // lanes past R follow the last
        u_raw[q] = static_cast<const T *>(a.u)[place[1][r] + k];
        dt_raw[q] = static_cast<const T *>(a.dt)[place[2][r] + k];
        if (USUAL || a.z) z_raw[q] = static_cast<const T *>(a.z)[place[3][r] + k];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        b[r].load(static_cast<const T *>(a.b) + place[4][r] + bc, whole);
        c[r].load(static_cast<const T *>(a.c) + place[5][r] + bc, whole);
    }
    load4(a.a + int64_t(k) * N + lane * 4, A);
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] *= kLog2e;
    const float bias = a.dt_bias ? a.dt_bias[k] : 0.f;
    const float skip = a.d ? a.d[k] : 0.f;
    float dt_mine[SHARE], u_mine[SHARE], gate_mine[SHARE];
#pragma unroll
    for (int q = 0; q < SHARE; ++q) {
        const float raw = to_float(dt_raw[q]);
        dt_mine[q] = USUAL || a.softplus ? softplus(raw, bias) : raw + bias;
        u_mine[q] = to_float(u_raw[q]);
        gate_mine[q] = USUAL || a.z ? silu(to_float(z_raw[q])) : 1.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int from = (threadIdx.x & 31) / P * P + r % P;
        const float dt = __shfl_sync(0xffffffffu, dt_mine[r / P % SHARE], from), u = __shfl_sync(0xffffffffu, u_mine[r / P % SHARE], from);
        float sum = 0.f;
        if (rows[r] >= 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[r][i] = fmaf(exp2_approx(dt * A[i]), h[r][i], dt * u * to_float(b[r].v[i]));
                sum = fmaf(to_float(c[r].v[i]), h[r][i], sum);
            }
            if (live)
                *reinterpret_cast<float4 *>(a.final_state + rows[r] + own) = make_float4(h[r][0], h[r][1], h[r][2], h[r][3]);
        }
#pragma unroll
        for (int o = P / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int64_t at = place[6][r];
        if (live && lane == r % P && at >= 0)
            static_cast<T *>(a.y)[at + k] = from_float<T>(rows[r] >= 0 ? fmaf(skip, u, sum) * gate_mine[r / P % SHARE] : 0.f);
    }
}

// Tokens of a chunk, 0 for whole sequences: the least of the estimated times, in ns.
// A warp alone takes `alone` for a token and a scheduler `turn` for a token of one
// of its warps, by the states of a lane (16: 178 and 118 measured; 8: 119 and 71);
// 64 states spread over four lanes cost half as much again.  Four CTAs an SM are
// resident (fp32 rows with 16 states: three, for their shared memory; not told
// apart), on the 148 SMs of a whole GPU: a stream of fewer takes the same chunks.
// Whole sequences last as long as the longest (the host does not know the lengths:
// of several, three times the mean is assumed); chunks take 1.75 of the passes (the
// first has no outputs), two launches more and the join, whose steps of 16 chunks
// are one trip to memory.  Measured, whole against chunks: 8 ragged prompts of 16384
// tokens x 4096 channels 1103 and 717 us, one of 8192 x 2048 1430 and 202 us, one of
// 300 x 1024 55 and 18 us, 58 ones of 14223 x 1736 even 197 and 308 us, ragged 380
// and 335.
int chunk_length(int tokens, int seqs, int channels, int states, int groups) {
    const int own = states < 16 ? states : 16, lanes = states > 16 ? states / 16 : 1;
    const int each = kScanThreads / (lanes < kScanThreads ? lanes : kScanThreads), per = (channels + groups - 1) / groups;
    const double columns = double(groups) * ((per + each - 1) / each), slow = states > 32 ? 1.5 : 1.0;
    const double turn = 5.9 * (own + 4) * slow, alone = (60 + 7.4 * own) * (slow > 1.0 ? 1.3 : 1.0);
    auto pass = [&](double length, double count) {
        const double ctas = columns * count, busy = ctas > 148 * 3 ? 4 : ctas > 148 * 2 ? 3 : ctas > 148 ? 2 : 1;
        const double one = 4000 + length * (alone > busy * turn ? alone : busy * turn), work = tokens * columns * turn / 148;
        return ctas <= 148 * 4 ? one : (work > one ? work : one) + 0.25 * length * alone;  // the rounds' end
    };
    const double mean = double(tokens) / seqs, longest = seqs == 1 || 3 * mean > tokens ? tokens : 3 * mean;
    const double together = pass(mean, seqs), whole = together > longest * alone ? together : longest * alone;
    double best = whole;
    int chosen = 0;
    for (int64_t length = 32; length < longest; length += 16 + length / 128 * 16) {
        const double count = double(tokens) / length + seqs;
        const double trips = (1 + longest / length / 16) * 1700, bytes = count * channels * states * 8 / 5000;
        const double cut = 8000 + (trips > bytes ? trips : bytes) + 1.75 * pass(length, count);
        if (cut < best) best = cut, chosen = int(length);
    }
    return chosen;
}

template <class T, int N>
cudaError_t launch_scan_as(const sq_scan_args &a, bool step, cudaStream_t s) {
    if (step) {
        constexpr int P = N / kPerLane;
        const unsigned grid = unsigned((int64_t(a.channels) * P + kScanThreads - 1) / kScanThreads);
        constexpr int64_t four = 4 * sizeof(T);
        auto fours = [&](const void *p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % four == 0 && stride % 4 == 0; };
        const bool whole = fours(a.b, a.b_stride) && fours(a.c, a.c_stride), usual = a.softplus && a.z;
        auto run = [&](auto kernel, int each) {
            const unsigned rows = unsigned((int64_t(a.num_seqs) + each - 1) / each);
            kernel<<<dim3(grid, rows < kGridRows ? rows : kGridRows, (rows + kGridRows - 1) / kGridRows), kScanThreads, 0, s>>>(a, whole);
        };
        // Few requests: one a lane, for the CTAs' number.
        if (int64_t(a.num_seqs) * grid < 148 * 16) usual ? run(scan_step_kernel<T, N, 1, true>, 1) : run(scan_step_kernel<T, N, 1, false>, 1);
        else usual ? run(scan_step_kernel<T, N, 4, true>, 4) : run(scan_step_kernel<T, N, 4, false>, 4);
        return cudaGetLastError();
    }
    const int per = a.channels / a.groups;
    constexpr int CH = ScanShape<T, N>::CH;
    const unsigned columns = unsigned(a.groups * ((per + CH - 1) / CH));
    Chunks chunks{};
    auto run = [&](auto kernel, int64_t parts, unsigned more) {
        constexpr int bytes = ScanShape<T, N>::kBytes;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        kernel<<<dim3(unsigned(parts) + more, columns), kScanThreads, bytes, s>>>(a, chunks, unsigned(parts));
        return cudaGetLastError();
    };
    if (a.workspace) chunks.length = chunk_length(a.tokens, a.num_seqs, a.channels, a.states, a.groups);
    const bool usual = a.softplus && a.z;
    if (!chunks.length) {
        const unsigned more = (37 + columns) / columns;
        return usual ? run(scan_kernel<T, N, kWhole, true>, a.num_seqs, more) : run(scan_kernel<T, N, kWhole, false>, a.num_seqs, more);
    }
    const int64_t count = a.tokens / chunks.length + a.num_seqs;
    chunks.state = static_cast<float *>(a.workspace);
    chunks.step_sum = chunks.state + count * a.channels * N;
    cudaError_t e = a.softplus ? run(scan_kernel<T, N, kChunkState, true>, count, 0) : run(scan_kernel<T, N, kChunkState, false>, count, 0);
    if (e != cudaSuccess) return e;
    join_kernel<<<dim3(unsigned(a.num_seqs) + 1, unsigned((int64_t(a.channels) * N + 255) / 256)), 256, 0, s>>>(a, chunks);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return usual ? run(scan_kernel<T, N, kChunkScan, true>, count, 0) : run(scan_kernel<T, N, kChunkScan, false>, count, 0);
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
    if (a.channels > (1 << 18) || a.groups > (1 << 14) || a.num_seqs > (1 << 30) || a.tokens > kMostTokens)
        return SQ_ERR_UNSUPPORTED;
    if (a.num_seqs == 0) return SQ_OK;
    if (!a.a || (a.tokens > 0 && (!a.u || !a.dt || !a.b || !a.c || !a.y))) return SQ_ERR_ARGUMENT;
    if (step ? !a.final_state : !a.cu_seqlens) return SQ_ERR_ARGUMENT;
    if (!a.slots && a.num_slots > 0 && a.num_slots < a.num_seqs) return SQ_ERR_CAPACITY;  // state row n of a smaller pool
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
    const int length = num_seqs ? sq::chunk_length(tokens, num_seqs, channels, states, groups) : 0;
    if (!length) return 0;
    return (int64_t(tokens / length) + num_seqs) * channels * (states + 1) * int64_t(sizeof(float));
}

extern "C" int32_t sq_selective_scan(const sq_scan_args *args, sq_stream_t stream) { return sq::scan_entry(args, false, stream); }

extern "C" int32_t sq_selective_scan_step(const sq_scan_args *args, sq_stream_t stream) {
    return sq::scan_entry(args, true, stream);
}
