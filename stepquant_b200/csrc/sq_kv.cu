// Appending keys and values to the paged 4-bit cache, keys rotated on the way, and
// reading them back.
//
// Eight neighbouring lanes hold a group of 64 channels of one token and head, eight
// channels each: the group's extremes are three shuffles away, and a lane's codes are
// one 32-bit word of the tile.  A code is that of the definition in exact arithmetic:
// fp32 finds it, with a bound on what its roundings may have changed, and groups where
// that reaches a border (a few in a thousand, more near position 0)
// are done again in 64 bits.  Append of 32768 tokens of 8 heads of 128: 169 us, 417
// instructions for a warp's 256 values at 2.2 a clock and SM (8192 tokens in one profiled session 57
// us; all in 64 bits 88), of which loads, stores and places take 140, the rotation 30 and the
// groups done again, which hold their CTA up, a quarter of the time.  No unit is full
// (adders 0.45): waits for loads, and stores of four bytes a lane, are what is left.  Read:
// 48 us, 3.6 TB/s, 135 instructions for a warp's 256 values at 2.0 a clock; its warps wait
// for words and pairs (four bytes a lane each) that follow a chain of boundaries, length and page.
#include "sq_kv.cuh"
#include "sq_rows.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kKvThreads = 256;
constexpr int kMostPerCta = 16;

struct Place {
    int64_t tile;  // byte offset of head 0's tile, -1: nowhere
    int64_t position;
    int token;
};

// Where new token i goes.
__device__ __forceinline__ Place place_of(const sq_kv_args &a, int i, int tile_bytes) {
    Place p{-1, 0, 0};
    if (a.num_seqs == 0) return p;
    int n = i;
    if (a.cu_seqlens) {
        if (i < sequence_range(a.cu_seqlens, 0, a.tokens).x || i >= sequence_range(a.cu_seqlens, a.num_seqs - 1, a.tokens).y)
            return p;
        int lo = 0, hi = a.num_seqs - 1;  // the last sequence that begins at or before i: the ones between are empty
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.cu_seqlens[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        n = lo;
        const int2 r = sequence_range(a.cu_seqlens, n, a.tokens);
        if (i >= r.y) return p;
        p.position = int64_t(a.lengths[n]) - r.y + i;
    } else {
        p.position = int64_t(a.lengths[n]) - 1;
    }
    p.tile = tile_at(a.page_table + n * a.table_stride, a.table_width, a.num_pages, p.position, a.page_size, a.heads, 0, tile_bytes,
                     a.status);
    p.token = int(p.position & (kTile - 1));
    return p;
}

// bf16 next to x towards -infinity, as its bits.
__device__ __forceinline__ uint32_t bf16_down(double x) {
    const uint32_t bits = __float_as_uint(__double2float_rd(x));
    return (bits & 0x80000000u ? bits + 0xFFFFu : bits) >> 16;
}
__device__ __forceinline__ uint32_t bf16_up(double x) { return bf16_down(-x) ^ 0x8000u; }
__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }

__device__ __forceinline__ double least8(double x, uint32_t lanes) {
#pragma unroll
    for (int i = 1; i < 8; i *= 2) x = fmin(x, __shfl_xor_sync(lanes, x, i));
    return x;
}

// Word and (s, m) of the group of which each of eight lanes holds x[0..7].
__device__ __forceinline__ void quantize(const double (&x)[8], uint32_t lanes, uint32_t &word, uint32_t &pair) {
    double low = x[0], high = -x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        low = fmin(low, x[i]);
        high = fmin(high, -x[i]);
        finite = finite && fabs(x[i]) <= 3.3895313892515355e38;  // the largest bf16; false for NaN
    }
    low = least8(low, lanes);
    high = -least8(high, lanes);
#pragma unroll
    for (int i = 1; i < 8; i *= 2) finite = __shfl_xor_sync(lanes, int(finite), i) && finite;
    if (!finite) {
        word = 0;
        pair = 0x7FC07FC0u;
        return;
    }
    const uint32_t m = bf16_down(low);
    const double base = bf16_value(m);
    const uint32_t s = bf16_up((high - base) / 15);
    const double step = s & 0x7FFF ? double(bf16_value(s)) : 1;
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= uint32_t(__double2int_rn((x[i] - base) / step)) << ((i >> 1) * 4 + (i & 1) * 16);
    pair = (s & 0x7FFF) | (m << 16);
}

// The same in fp32 of x[0..7], each within `off` of the value that is meant (0: exact).  False in all eight
// lanes where a result may be another in exact arithmetic.
__device__ __forceinline__ bool quantize_fast(const float (&x)[8], float off, uint32_t lanes, uint32_t &word, uint32_t &pair) {
    float low = fminf(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5])), high = fmaxf(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]));
    low = min3(low, x[6], x[7]);
    high = max3(high, x[6], x[7]);
#pragma unroll
    for (int i = 1; i < 8; i *= 2) {
        low = fminf(low, __shfl_xor_sync(lanes, low, i));
        high = fmaxf(high, __shfl_xor_sync(lanes, high, i));
        off = fmaxf(off, __shfl_xor_sync(lanes, off, i));
    }
    auto down = [](float y) {
        const uint32_t bits = __float_as_uint(y);
        return (bits & 0x80000000u ? bits + 0xFFFFu : bits) & 0xFFFF0000u;
    };
    // The minimum: on one side of a border with all that it may be.
    const uint32_t m_bits = down(low);
    bool sure = off == 0.f || (down(low - 1.25f * off) == m_bits && down(low + 1.25f * off) == m_bits);
    const float m = __uint_as_float(m_bits);
    // The scale: s the least bf16 with 15 s >= d.  15 s has 12 bits.
    const float d = high - m;
    sure = sure && (off != 0.f || (d + m == high && high - d == m)) && d < 1e38f && d > 1e-30f && fmaxf(high, -low) < 3e38f;
    uint32_t s_bits = (__float_as_uint(d * (1.f / 15.f)) + 0xFFFFu) & 0xFFFF0000u;  // or one above or below
    if (15.f * __uint_as_float(s_bits - 0x10000u) >= d) s_bits -= 0x10000u;
    if (15.f * __uint_as_float(s_bits) < d) s_bits += 0x10000u;
    const float s = __uint_as_float(s_bits), slack = 2.f * off + d * 0x1p-20f, least = off == 0.f ? 0.f : slack;
    sure = sure && 15.f * s - d >= least && d - 15.f * __uint_as_float(s_bits - 0x10000u) > least;
    // Whole numbers near 1.5 * 2^23 have theirs in the last bits; a code whose rest is not within the slack of half a
    // step is the right one.
    constexpr float kWhole = 12582912.f;
    const float per = reciprocal_approx(s), clear = 0.5f * (s - slack);
    float farthest = 0.f;
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float e = x[i] - m, near = fmaf(e, per, kWhole), rest = fmaf(kWhole - near, s, e);
        const float e1 = x[i + 1] - m, near1 = fmaf(e1, per, kWhole), rest1 = fmaf(kWhole - near1, s, e1);
        farthest = max3_or_nan(farthest, fabsf(rest), fabsf(rest1));  // not a number where a value is not finite
        // Codes i and i + 1 to bits 2 i and 2 i + 16, by multiplications (the adders are the busier ones).
        word += (__float_as_uint(near) - 0x4B400000u) * (1u << (2 * i)) + (__float_as_uint(near1) - 0x4B400000u) * (1u << (2 * i + 16));
    }
    bool all = farthest < clear;
    if (!all && off == 0.f) {  // exact values: ties, to the even code, and their neighbours
        all = true;
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = x[i] - m, near = fmaf(e, per, kWhole), rest = fmaf(kWhole - near, s, e);
            const float beyond = 2.f * fabsf(rest) - s;  // above 0: the next; 0: a tie
            const uint32_t code = __float_as_uint(near) - 0x4B400000u;
            const bool next = bool(beyond > 0.f) | (bool(beyond == 0.f) & bool(code & 1));
            word += (code + (next ? (rest > 0.f ? 1u : ~0u) : 0u)) << ((i >> 1) * 4 + (i & 1) * 16);
            all &= bool(fabsf(rest) < clear) | (bool(e + m == x[i]) & bool(x[i] - e == m));
        }
    }
    sure = sure && all;
    pair = (s_bits >> 16) | m_bits;
    return (__ballot_sync(lanes, sure) & lanes) == lanes;
}

template <class T>
__device__ __forceinline__ void load8(const T *p, bool wide, T (&x)[8]) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i) reinterpret_cast<uint4 *>(x)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}

// Channels c..c + 7 of a key in 64 bits, rotated.
template <class T>
__device__ __noinline__ void turn_exactly(const sq_kv_args &a, const T *k, int c, int64_t position, double (&x)[8]) {
    const int half = a.turned / 2;
    for (int e = 0; e < 8; ++e) {
        const int at = c + e;
        x[e] = to_float(k[at]);
        if (at >= a.turned) continue;
        const int f = a.interleaved ? at / 2 : at < half ? at : at - half;
        const bool second = a.interleaved ? at & 1 : at >= half;
        const double other = to_float(k[a.interleaved ? at ^ 1 : second ? at - half : at + half]);
        // The nearest quarter of a turn goes first: what is left of an angle near it keeps its bits in 64.
        const uint64_t phase = uint64_t(phase_of(position, a.frequencies[f])), quarters = (phase + (uint64_t(1) << 61)) >> 62;
        double sin, cos;
        sincospi(double(int64_t(phase - (quarters << 62))) * 0x1p-63, &sin, &cos);
        if (quarters & 1) {
            const double other_one = cos;
            cos = -sin;
            sin = other_one;
        }
        cos *= quarters & 2 ? -a.magnitude : a.magnitude;
        sin *= quarters & 2 ? -a.magnitude : a.magnitude;
        x[e] = second ? other * sin + x[e] * cos : x[e] * cos - other * sin;
    }
}

template <class T, int D>
__global__ void __launch_bounds__(kKvThreads, 4) kv_append_kernel(sq_kv_args a, int per_cta, bool k_wide, bool v_wide) {
    using Tile = KvTile<D>;
    constexpr int kLanes = D / 8;  // of one head's keys or values
    extern __shared__ __align__(16) float2 table[];  // [per_cta][turned / 2] (cos, sin), times the magnitude
    __shared__ Place places[kMostPerCta];
    const int64_t first = int64_t(blockIdx.x) * per_cta;
    const int count = int(min(int64_t(per_cta), a.tokens - first)), half = a.turned / 2;
    if (int(threadIdx.x) < count) {
        Place p = place_of(a, int(first) + threadIdx.x, Tile::kBytes);
        if (a.positions) p.position = position_at(a.positions, a.position_dtype, first + threadIdx.x);
        places[threadIdx.x] = p;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count * half; i += kKvThreads) {
        const int t = i / half, f = i - t * half;
        float sin, cos;
        sincospif(float(int32_t(phase_of(places[t].position, a.frequencies[f]) >> 32)) * 0x1p-31f, &sin, &cos);
        table[i] = make_float2(a.magnitude * cos, a.magnitude * sin);
    }
    __syncthreads();
    const int lanes = a.heads * 2 * kLanes;  // of a token, keys first: a multiple of 16
    const int64_t head_bytes = int64_t(a.page_size / kTile) * Tile::kBytes;
    const uint32_t group_lanes = 0xFFu << (threadIdx.x & 24);
    const bool pairs_wide = k_wide && half % 8 == 0;
    // What a rotated channel is off by at most, in units of 2^-24 (|x1| + |x2|): sine and cosine by pi / 2 (their
    // argument in half turns is rounded to fp32), 1 (the functions) and 1/2 (the magnitude's product), then the
    // products and their sum by 1/2 each; 4.1 in all, and |x1| + |x2| is at most twice the larger.
    const float turn_off = 0x1.1p-21f * fabsf(a.magnitude);
    // Threads are [token][lane] where a token's lanes are fewer than them.
    const int t_step = max(1, kKvThreads / lanes), t0 = int(threadIdx.x) / lanes < t_step ? int(threadIdx.x) / lanes : 0;
    if (lanes < kKvThreads && int(threadIdx.x) >= t_step * lanes) return;
    for (int rest = int(threadIdx.x) - t0 * lanes; rest < lanes; rest += kKvThreads) {
        const int values = 2 * rest >= lanes, head = (values ? rest - lanes / 2 : rest) / kLanes, lane = rest % kLanes;
        const int c = lane * 8, group = lane >> 3, w = lane & 7;
        const int64_t stride = values ? a.v_stride : a.k_stride;
        const T *from = values ? static_cast<const T *>(a.v) + head * a.v_head_stride : static_cast<const T *>(a.k) + head * a.k_head_stride;
        from += (first + t0) * stride;
        uint8_t *const to = a.data + head * head_bytes;
        const bool wide = values ? v_wide : k_wide;
        for (int t = t0; t < count; t += t_step, from += t_step * stride) {
        const Place &p = places[t];
        if (p.tile < 0) continue;
        alignas(16) T raw[8];
        float x[8], off = 0.f;
        load8(from + c, wide, raw);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_float(raw[e]);
        if (!values && c < a.turned) {
            const float2 *cs = table + t * half;
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    if (c + e < a.turned) {
                        const float2 z = cs[(c + e) / 2];
                        const float u = x[e], w = x[e + 1];
                        off = max3(off, fabsf(u), fabsf(w));
                        x[e] = u * z.x - w * z.y;
                        x[e + 1] = u * z.y + w * z.x;
                    }
                }
            } else if (pairs_wide) {
                const bool upper = c >= half;
                const int f = upper ? c - half : c;
                alignas(16) T other[8];
                load8(from + (upper ? f : c + half), true, other);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 z = cs[f + e];
                    const float w = to_float(other[e]);
                    off = max3(off, fabsf(x[e]), fabsf(w));
                    x[e] = x[e] * z.x + (upper ? w : -w) * z.y;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (c + e < a.turned) {
                        const bool upper = c + e >= half;
                        const int f = upper ? c + e - half : c + e;
                        const float w = to_float(from[upper ? f : c + e + half]);
                        const float2 z = cs[f];
                        off = max3(off, fabsf(x[e]), fabsf(w));
                        x[e] = x[e] * z.x + (upper ? w : -w) * z.y;
                    }
                }
            }
            off *= turn_off;
        }
        uint32_t word, pair;
        if (!quantize_fast(x, off, group_lanes, word, pair)) {
            double exact[8];
            if (values || c >= a.turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) exact[e] = to_float(raw[e]);
            } else {
                turn_exactly(a, from, c, p.position, exact);
            }
            quantize(exact, group_lanes, word, pair);
        }
        uint8_t *tile = to + p.tile;
        *reinterpret_cast<uint32_t *>(tile + (values ? Tile::value_word(p.token, group, w) : Tile::key_word(p.token, group, w))) = word;
        if (w == 0) *reinterpret_cast<uint32_t *>(tile + Tile::pair(values, p.token, group)) = pair;
        }
    }
}

template <class T, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(sq_kv_args a, int per_cta) {
    using Tile = KvTile<D>;
    constexpr int kLanes = D / 8;
    __shared__ Place places[kMostPerCta];
    const int64_t first = int64_t(blockIdx.x) * per_cta;
    const int count = int(min(int64_t(per_cta), a.tokens - first));
    if (int(threadIdx.x) < count) places[threadIdx.x] = place_of(a, int(first) + threadIdx.x, Tile::kBytes);
    __syncthreads();
    const int lanes = a.heads * 2 * kLanes;
    const int64_t head_bytes = int64_t(a.page_size / kTile) * Tile::kBytes;
    int t = int(threadIdx.x) / lanes, rest = int(threadIdx.x) - t * lanes;
    const int t_step = kKvThreads / lanes, rest_step = kKvThreads - t_step * lanes;
#pragma unroll 4
    for (; t < count; t += t_step, rest += rest_step, t += rest >= lanes, rest -= rest >= lanes ? lanes : 0) {
        const int values = 2 * rest >= lanes, head = (values ? rest - lanes / 2 : rest) / kLanes, lane = rest % kLanes;
        const Place &p = places[t];
        const int group = lane >> 3, w = lane & 7;
        uint32_t word = 0, pair = 0;
        if (p.tile >= 0) {
            const uint8_t *tile = a.data + p.tile + head * head_bytes;
            word = __ldg(reinterpret_cast<const uint32_t *>(tile + (values ? Tile::value_word(p.token, group, w) : Tile::key_word(p.token, group, w))));
            pair = __ldg(reinterpret_cast<const uint32_t *>(tile + Tile::pair(values, p.token, group)));
        }
        const float s = bf16_value(pair & 0xFFFF), m = bf16_value(pair >> 16);
        alignas(16) T x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = from_float<T>(fmaf(s, float(word >> ((e >> 1) * 4 + (e & 1) * 16) & 15), m));
        T *out = values ? static_cast<T *>(a.v) + (first + t) * a.v_stride + head * a.v_head_stride
                        : static_cast<T *>(a.k) + (first + t) * a.k_stride + head * a.k_head_stride;
#pragma unroll
        for (int e = 0; e < int(sizeof(T)) / 2; ++e) reinterpret_cast<uint4 *>(out + lane * 8)[e] = reinterpret_cast<uint4 *>(x)[e];
    }
}

template <class T, int D>
cudaError_t launch_kv(const sq_kv_args &a, bool append, cudaStream_t s) {
    int per_cta = kMostPerCta;
    while (per_cta > 1 && (int64_t(a.tokens) + per_cta - 1) / per_cta < 148 * 2) per_cta /= 2;
    const unsigned grid = unsigned((int64_t(a.tokens) + per_cta - 1) / per_cta);
    auto wide = [&](const void *p, int64_t token, int64_t head) {
        constexpr int n = 16 / sizeof(T);
        return aligned16(p) && token % n == 0 && head % n == 0;
    };
    const bool k_wide = wide(a.k, a.k_stride, a.k_head_stride), v_wide = wide(a.v, a.v_stride, a.v_head_stride);
    if (append) {
        kv_append_kernel<T, D><<<grid, kKvThreads, size_t(per_cta) * (a.turned / 2) * sizeof(float2), s>>>(a, per_cta, k_wide, v_wide);
    } else {
        if (!k_wide || !v_wide) return cudaErrorInvalidValue;
        kv_read_kernel<T, D><<<grid, kKvThreads, 0, s>>>(a, per_cta);
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_kv(const sq_kv_args &a, bool append, cudaStream_t s) {
    switch (a.dim) {
        case 64: return launch_kv<T, 64>(a, append, s);
        case 128: return launch_kv<T, 128>(a, append, s);
        default: return launch_kv<T, 256>(a, append, s);
    }
}

int32_t kv_entry(const sq_kv_args *args, bool append, sq_stream_t stream) {
    if (!args) return SQ_ERR_ARGUMENT;
    const sq_kv_args &a = *args;
    if (a.tokens < 0 || a.num_seqs < 0 || a.table_width < 0 || a.num_pages < 0 || a.heads < 1 || a.turned < 0) return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16 || !(fabsf(a.magnitude) < INFINITY)) return SQ_ERR_ARGUMENT;
    if (a.dim != 64 && a.dim != 128 && a.dim != 256) return SQ_ERR_UNSUPPORTED;
    if (a.page_size < kTile || a.page_size % kTile || a.turned % 2 || a.turned > a.dim || a.table_stride < 0) return SQ_ERR_SHAPE;
    if (a.k_stride < 0 || a.k_head_stride < 0 || a.v_stride < 0 || a.v_head_stride < 0 || !aligned16(a.data)) return SQ_ERR_SHAPE;
    if (a.heads > 4096 || a.page_size > 65536 || a.tokens > kMostTokens || a.num_seqs > (1 << 30)) return SQ_ERR_UNSUPPORTED;
    if (int64_t(a.table_width) * a.page_size > kMostTokens) return SQ_ERR_UNSUPPORTED;  // positions are ints
    if (!a.cu_seqlens && a.tokens != a.num_seqs) return SQ_ERR_ARGUMENT;
    if (a.tokens == 0) return SQ_OK;
    if (!a.k || !a.v || (a.num_seqs && (!a.lengths || (a.table_width && !a.page_table) || (a.num_pages && !a.data)))) return SQ_ERR_ARGUMENT;
    if (append && a.turned && !a.frequencies) return SQ_ERR_ARGUMENT;
    if (!append && (!aligned16(a.k) || !aligned16(a.v) || (a.k_stride | a.k_head_stride | a.v_stride | a.v_head_stride) % 8)) return SQ_ERR_SHAPE;
    if (append && a.num_seqs == 0) return SQ_OK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SQ_F32    ? launch_kv<float>(a, append, s)
                          : a.dtype == SQ_BF16 ? launch_kv<__nv_bfloat16>(a, append, s)
                                               : launch_kv<__half>(a, append, s);
    return e == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}

}  // namespace
}  // namespace sq

extern "C" int32_t sq_kv_append(const sq_kv_args *args, sq_stream_t stream) { return sq::kv_entry(args, true, stream); }

extern "C" int32_t sq_kv_read(const sq_kv_args *args, sq_stream_t stream) { return sq::kv_entry(args, false, stream); }
