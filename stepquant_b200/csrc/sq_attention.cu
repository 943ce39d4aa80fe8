// Attention over the paged 4-bit cache (sq_kv.cu):
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max)
//
// with k_j = m + s c for each group of 64 channels.  Scale and minimum of a key leave
// the product, q . k = sum over groups of s (q . c) + m sum(q), and those of a value go
// to its weight, p v = (p s) c + p m, so the tensor cores work on the codes, which 16
// bits hold exactly.
//
// Few rows (rows_kernel): mma.sync with tokens (scores) or channels (values) as the 16
// rows and eight query rows as columns; a warp's fragments are the tile's words with a
// shift and a mask.  The products are a fifth of the tensor pipe's time: with eight columns
// tcgen05 would idle as much and want the codes unpacked into shared memory first.
// 256 ragged requests of up to 8192 tokens (1.3 GB) take 357 us, 3.7 TB/s: 444 instructions
// a tile of 16 tokens and 2304 bytes (64 masks, 48 shifts, 32 differences, 32 products, the
// rest scales, exponentials and waits) at 2.5 a clock and SM.  No unit is full (adders 0.56,
// DRAM 0.55 of the copy rate): sixteen warps an SM, at 128 registers each, do not hide what
// each instruction waits for the one before.
//
// Sums are fp32, but the tensor cores cut theirs off: up to 6e-9 of a sum a token (8e-4 at
// 131072 tokens of equal weights and values), in both kernels.  So codes are summed about a
// middle.
#include "sq_kv.cuh"
#include "sq_rows.cuh"
#include "sq_tc.cuh"
#include "sq_vec.cuh"

namespace sq {

cudaError_t launch_prompt_attention(const sq_kv_attention_args &a, int few_rows, cudaStream_t s);  // sq_attention_prompt.cu

namespace {

constexpr int kWarps = 8, kAttnThreads = 32 * kWarps;
constexpr int kMostCtas = 320;
constexpr int kUnit = 32;             // tokens that a warp takes at a time: two tiles of the cache
constexpr int kLeastUnits = kWarps;   // of a CTA
constexpr int kItemUnits = 16;        // what the start and the end of an item cost a CTA
constexpr float kNone = -3.402823466e38f;  // a maximum over nothing
constexpr int kFewRows = 32;

// ---------------------------------------------------------------------------
// fragments
// ---------------------------------------------------------------------------
constexpr float kMiddle = 8.f;  // values' codes are multiplied as c - 8

template <class T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
    // Weights of bf16 queries are bf16 too: half a step of 2^-9, the size of an output's own rounding (256 requests: off
    // by 2.1e-3 of the outputs' norm in all, of which that is 1.7e-3).  f16 weights would need what f16 queries do about
    // p s (below; 403 us for 357) and more, as bf16 values go far beyond f16 either way.
    static constexpr float kHeld = 128.f;  // pair() is c + this: a bf16 with c in its last bits
    __device__ static __forceinline__ uint32_t pair(uint32_t w) { return and_or(w, 0x000F000Fu, 0x43004300u); }
    // c - 8, for sums over many tokens: the tensor cores cut sums off, and those of 128 + c, 136 times the weights' sum
    // taken off at the end, were 4 % of the outputs' norm off where a warp had 4096 tokens (256 requests 353 -> 338 us, too).
    __device__ static __forceinline__ uint32_t centred(uint32_t w, uint32_t) {
        const uint32_t x = pair(w), base = 0x43084308u;
        const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(x), reinterpret_cast<const __nv_bfloat162 &>(base));
        return reinterpret_cast<const uint32_t &>(r);
    }
    __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    __device__ static __forceinline__ float2 unpack(uint32_t x) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
    }
    __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static constexpr float kLag = 8.f;
    static constexpr bool kNarrow = false;  // p s has fp32's range
};
template <>
struct Codes<__half> {
    static constexpr float kHeld = -kMiddle;  // f16 with c in their last bits are 1024 + c, too far from c to leave it in
    __device__ static __forceinline__ uint32_t centred(uint32_t w, uint32_t base) {
        const uint32_t x = and_or(w, 0x000F000Fu, 0x64006400u);
        const __half2 r = __hsub2(reinterpret_cast<const __half2 &>(x), reinterpret_cast<const __half2 &>(base));
        return reinterpret_cast<const uint32_t &>(r);
    }
    __device__ static __forceinline__ uint32_t pair(uint32_t w) { return centred(w, 0x64086408u); }
    __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    __device__ static __forceinline__ float2 unpack(uint32_t x) { return __half22float2(reinterpret_cast<const __half2 &>(x)); }
    __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    // p s has f16's range only, so what weights are taken against depends on p s: a row's reference R, p = 2^(score - R),
    // rises where a p s is above kMostWeight, to bring that one to 2^8 .. 2^9 (what rounding loses of the others is then
    // 2^-33 of the row's largest), or a p above 2^kMostPower, to bring it to 2^kLag (the scales are tiny then, and
    // 2^-25 over 2^kLag is far below what an f16 output holds).
    static constexpr bool kNarrow = true;
    static constexpr float kLag = 24.f, kMostPower = 32.f, kMostWeight = 61440.f;
};

// Transpose of an 8 x 8 matrix of 16-bit values, two of row lane / 4 in each lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ float pair_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float pair_min(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

// ---------------------------------------------------------------------------
// work: units of 32 tokens in the order (sequence, kv head, block of rows, unit), each item's after
// kItemUnits for its start and end, cut into equal spans of consecutive ones, a span to a CTA
// ---------------------------------------------------------------------------
struct Sequence {
    int first, count;   // new tokens
    int length;         // tokens that the page table reaches
    int64_t before;     // position of the first new token
    int seen_from;      // first position that any of them sees, `length` if none does
    int unit, units;    // units that any of them sees: one at least
    int blocks;         // of rows (token, query head of the kv head)
    int64_t cost;
};

template <int ROWS>
__device__ __forceinline__ Sequence sequence(const sq_kv_attention_args &a, int most_rows, int n, bool report) {
    Sequence s;
    const int2 r = a.cu_seqlens ? sequence_range(a.cu_seqlens, n, a.tokens) : make_int2(n, n + 1);
    s.first = r.x;
    s.count = r.y - r.x;
    const int length = a.lengths[n];
    const int64_t most = int64_t(a.table_width) * a.page_size;
    if (report && s.count > 0 && length > most) flag(a.status, SQ_STATUS_SLOT_RANGE);
    s.length = int(max(int64_t(0), min(int64_t(length), most)));
    s.before = int64_t(length) - s.count;
    const int64_t start = a.window > 0 ? max(int64_t(0), s.before - a.window + 1) : 0;
    s.seen_from = int(min(start, int64_t(s.length)));
    s.unit = s.seen_from / kUnit;
    s.units = max(1, int((int64_t(s.length) + kUnit - 1) / kUnit) - s.unit);
    const int64_t rows = int64_t(s.count) * (a.q_heads / a.heads);
    s.blocks = rows > most_rows ? 0 : int((rows + ROWS - 1) / ROWS);
    s.cost = int64_t(s.blocks) * a.heads * (kItemUnits + s.units);
    return s;
}

// a / b of numbers that seldom need 64 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return uint64_t(a | b) >> 32 ? a / b : int64_t(uint32_t(a) / uint32_t(b));
}

struct Span {
    int64_t begin, end, per;  // in units
    int sequence;             // that begin lies in
    int64_t offset;           // of begin in it
};

// This CTA's span (begin = end: none).  Every thread of the CTA calls it.
template <int ROWS>
__device__ __forceinline__ Span span_of(const sq_kv_attention_args &a, int most_rows, bool report) {
    __shared__ int64_t warp_sums[kWarps];
    __shared__ int64_t found_offset;
    __shared__ int found;
    const int each = (a.num_seqs + kAttnThreads - 1) / kAttnThreads;
    const int from = min(int(threadIdx.x) * each, a.num_seqs), to = min(from + each, a.num_seqs);
    int64_t mine = 0;
    for (int n = from; n < to; ++n) mine += sequence<ROWS>(a, most_rows, n, report).cost;
    int64_t sum = mine;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
        const int64_t other = __shfl_up_sync(~0u, sum, i);
        if (lane >= i) sum += other;
    }
    if (lane == 31) warp_sums[warp] = sum;
    if (threadIdx.x == 0) found = 0, found_offset = 0;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) sum += warp_sums[w];
        total += warp_sums[w];
    }
    Span s;
    s.per = max(int64_t(kLeastUnits), quotient(total + gridDim.x - 1, gridDim.x));
    s.begin = min(total, s.per * blockIdx.x);
    s.end = min(total, s.begin + s.per);
    int64_t at = sum - mine;
    if (s.begin < s.end && at <= s.begin && s.begin < sum) {
        for (int n = from; n < to; ++n) {
            const int64_t cost = sequence<ROWS>(a, most_rows, n, false).cost;
            if (s.begin < at + cost) {
                found = n;
                found_offset = s.begin - at;
                break;
            }
            at += cost;
        }
    }
    __syncthreads();
    s.sequence = found;
    s.offset = found_offset;
    return s;
}

template <class T>
__device__ __forceinline__ T *output_row(const sq_kv_attention_args &a, const Sequence &s, int head, int row) {
    const int group = a.q_heads / a.heads;
    return static_cast<T *>(a.out) + ((int64_t(s.first) + row / group) * a.q_heads + head * group + row % group) * a.dim;
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
template <int D, int NT>
struct RowsShape {
    using Tile = KvTile<D>;
    static constexpr int kRows = 8 * NT;
    static constexpr int kStages = D == 64 ? 3 : 2;  // units
    static constexpr int kStage = 2 * Tile::kBytes, kRing = kStages * kStage;  // of a warp
    static constexpr int kMergeRow = D + 4;                       // floats
    static constexpr int kMerge = kRows * kMergeRow * 4;          // of a warp
    static constexpr int kPart = kRows * D + 2 * kRows;           // floats of a part: sums, maxima, weights' sums
    static constexpr int kShared = kWarps * (kRing + kMerge);
    static_assert(kRing % 16 == 0 && kMerge % 16 == 0 && Tile::kBytes % 16 == 0, "copies and sums are aligned");
};

// The units of one item that lie in a CTA's span.
struct Segment {
    int sequence, head, block;
    int first, tokens, length;  // the sequence's new tokens, tokens that it holds
    int64_t before;             // position of its first new token
    int seen_from;              // first position that any of them sees
    int unit, count;            // first unit, units; none: the span is over
    bool whole;                 // the item's units
};

// Where in its span a CTA is.
struct Cursor {
    Sequence s;
    int64_t at;
    int n, head, block, begin;  // begin: what lies before in the item
};

template <int ROWS>
__device__ __forceinline__ void next_segment(const sq_kv_attention_args &a, int most_rows, int64_t end, Cursor &c, Segment &g) {
    g.count = 0;
    while (c.at < end && g.count == 0) {
        if (c.begin >= kItemUnits + c.s.units) {
            c.begin = 0;
            if (++c.block >= c.s.blocks) {
                c.block = 0;
                ++c.head;
            }
        }
        while (c.head >= a.heads || c.s.cost == 0) {  // on to the next sequence with new tokens: there is one, as at < end
            c.s = sequence<ROWS>(a, most_rows, ++c.n, false);
            c.head = c.block = c.begin = 0;
        }
        const int step = int(min(end - c.at, int64_t(kItemUnits + c.s.units - c.begin)));
        const int first = max(0, c.begin - kItemUnits);
        c.at += step;
        c.begin += step;
        g.count = max(0, c.begin - kItemUnits) - first;  // none: the span ends with the item's start
        g.unit = c.s.unit + first;
    }
    g.sequence = c.n, g.head = c.head, g.block = c.block;
    g.first = c.s.first, g.tokens = c.s.count, g.length = c.s.length, g.before = c.s.before, g.seen_from = c.s.seen_from;
    g.whole = g.count == c.s.units;
}

template <int N>
struct Words;
template <>
struct Words<1> { using type = uint32_t; };
template <>
struct Words<2> { using type = uint2; };
template <>
struct Words<4> { using type = uint4; };
template <int N>
__device__ __forceinline__ void load_words(const uint8_t *from, uint32_t (&w)[N]) {
    *reinterpret_cast<typename Words<N>::type *>(w) = *reinterpret_cast<const typename Words<N>::type *>(from);
}

template <class T, int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 && D <= 128 ? 2 : 1) rows_kernel(sq_kv_attention_args a, int most_rows) {
    using Shape = RowsShape<D, NT>;
    using Tile = KvTile<D>;
    using C = Codes<T>;
    constexpr int kGroups = Tile::kGroups, kRows = Shape::kRows, kStages = Shape::kStages;
    extern __shared__ __align__(128) uint8_t rings[];
    __shared__ uint64_t bars[kWarps][kStages];
    __shared__ float row_max[kWarps][kRows], row_sum[kWarps][kRows];
    __shared__ Segment segments[4];  // this one, the next (whose first units are requested meanwhile) and the one after
    __shared__ Cursor cursor;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t *const ring = rings + warp * Shape::kRing;
    float *const merge = reinterpret_cast<float *>(rings + kWarps * Shape::kRing);
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) tc::bar_init(&bars[warp][i], 1);
        tc::bar_init_fence();
    }
    if (a.cu_seqlens)
        clear_outside(a.out, int64_t(a.q_heads) * D * sizeof(T), a.cu_seqlens, a.num_seqs, a.tokens, blockIdx.x, gridDim.x);
    const Span span = span_of<kRows>(a, most_rows, blockIdx.x == 0);
    const int group = a.q_heads / a.heads, page_tiles = a.page_size / kTile;
    const float to_log2 = a.scale * kLog2e, lag = C::kLag / to_log2;
    const int64_t head_bytes = int64_t(page_tiles) * Tile::kBytes;
    // Queries on their way to L2: two lines of 128 bytes a lane at most.
    auto fetch_rows = [&](const Segment &s) {
        constexpr int kLines = (D * 2 + 127) / 128;
        for (int i = lane; i < kRows * kLines && s.count; i += 32) {
            const int row = s.block * kRows + i / kLines;
            if (row < s.tokens * group) {
                const int token = row / group;
                const T *from = static_cast<const T *>(a.q) + (int64_t(s.first) + token) * a.q_stride +
                                int64_t(s.head * group + row - token * group) * a.q_head_stride + i % kLines * 64;
                asm volatile("prefetch.global.L2 [%0];\n" ::"l"(from));
            }
        }
    };
    if (warp == 0) {
        if (lane == 0) {
            Cursor c;
            c.at = span.begin;
            c.n = span.sequence;
            c.s = sequence<kRows>(a, most_rows, min(c.n, a.num_seqs - 1), false);
            const int item = c.s.cost ? int(quotient(span.offset, kItemUnits + c.s.units)) : 0;
            c.begin = c.s.cost ? int(span.offset - int64_t(item) * (kItemUnits + c.s.units)) : 0;
            c.head = c.s.cost ? item / c.s.blocks : 0;
            c.block = c.s.cost ? item % c.s.blocks : 0;
            next_segment<kRows>(a, most_rows, span.end, c, segments[0]);
            next_segment<kRows>(a, most_rows, span.end, c, segments[1]);
            cursor = c;
        }
        __syncwarp();
        fetch_rows(segments[0]);
        fetch_rows(segments[1]);
    }
    __syncthreads();

    // This warp's units of a segment are number warp, warp + 8, ...; its ring holds those of this segment and then
    // of the next.
    auto units_of = [&](const Segment &s) { return (s.count - warp + kWarps - 1) / kWarps; };
    int request_stage = 0;
    int64_t places = -1;  // lane 2 i + h: byte offset of tile h of unit i, modulo 16, of the segment that is requested; -1: none
    uint32_t missing = 0; // by stage, two bits: whether there was no tile to load; from kArmed on, one: not waited for yet
    constexpr int kArmed = 16;
    auto request = [&](const Segment &s, int i) {
        if ((i & 15) == 0) {
            places = -1;
            const int unit = warp + (i + lane / 2) * kWarps, tile = (s.unit + unit) * 2 + (lane & 1), index = tile / page_tiles;
            // A unit's tile past the sequence's end or in front of every row's window is not looked up: the table may hold
            // anything there.
            if (unit < s.count && index < a.table_width && tile * kTile < s.length && (tile + 1) * kTile > s.seen_from) {
                const int page = a.page_table[s.sequence * a.table_stride + index];
                if (page >= a.num_pages) flag(a.status, SQ_STATUS_SLOT_RANGE);
                else if (page > 0) places = (int64_t(page) * a.heads + s.head) * head_bytes + int64_t(tile - index * page_tiles) * Tile::kBytes;
            }
        }
        // Lanes 0 and 1 fetch a tile each.
        const int64_t place = __shfl_sync(~0u, places, 2 * (i & 15) + (lane & 1));
        const uint32_t none = __ballot_sync(~0u, place < 0) & 3;
        missing = (missing & ~(3u << 2 * request_stage)) | none << 2 * request_stage | 1u << (kArmed + request_stage);
        uint64_t *const bar = &bars[warp][request_stage];
        if (lane == 0) tc::bar_expect(bar, (none == 0 ? 2 : none == 3 ? 0 : 1) * Tile::kBytes);
        if (lane < 2 && place >= 0)
            tc::bulk_load(ring + request_stage * Shape::kStage + lane * Tile::kBytes, a.data + place, Tile::kBytes, bar);
        request_stage = request_stage + 1 == kStages ? 0 : request_stage + 1;
    };
    int ahead = 0;  // units of the next segment that were requested
    int stage = 0;
    uint32_t phase = 0;
    bool gave_up = false;  // of the whole warp: it waits for no more units and requests none
    for (int number = 0; segments[number & 3].count; ++number) {
        const Segment &here = segments[number & 3];  // for what is seldom read
        const Segment s = here;
        const Segment &next = segments[(number + 1) & 3];
        const int mine = units_of(s);
        for (int i = ahead; i < min(mine, kStages) && !gave_up; ++i) request(here, i);
        ahead = min(mine, max(ahead, kStages));
        if (warp == (number & (kWarps - 1))) {
            if (lane == 0) {
                Cursor c = cursor;
                next_segment<kRows>(a, most_rows, span.end, c, segments[(number + 2) & 3]);
                cursor = c;
            }
            __syncwarp();
            fetch_rows(segments[(number + 2) & 3]);
        }

        // Query rows as the product's second operand: row g's channels 16 t + 0..15 of each group.
        uint32_t q[NT][kGroups][8];
        float q_sum[NT][kGroups][2];  // of rows 2 t and 2 t + 1: the groups' sums
        int place[NT][2];     // their positions, which may lie past the table
        const int row0 = s.block * kRows, rows = s.tokens * group;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int row = row0 + j * 8 + g;
            const bool live = row < rows;
            const int token = live ? row / group : 0, head = live ? row - token * group : 0;
            const T *from = static_cast<const T *>(a.q) + (int64_t(s.first) + token) * a.q_stride + int64_t(s.head * group + head) * a.q_head_stride + 16 * t;
#pragma unroll
            for (int b = 0; b < kGroups; ++b) {
                const uint4 x = reinterpret_cast<const uint4 *>(from + b * kGroup)[0], y = reinterpret_cast<const uint4 *>(from + b * kGroup)[1];
                const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    q[j][b][i] = live ? w[i] : 0;
                    const float2 v = C::unpack(q[j][b][i]);
                    sum += v.x + v.y;
                }
                sum += __shfl_xor_sync(~0u, sum, 1);
                sum += __shfl_xor_sync(~0u, sum, 2);  // of row g; rows 2 t, 2 t + 1 are in lanes 8 t, 8 t + 4
                q_sum[j][b][0] = __shfl_sync(~0u, sum, 8 * t);
                q_sum[j][b][1] = __shfl_sync(~0u, sum, 8 * t + 4);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = row0 + j * 8 + 2 * t + e;
                place[j][e] = r < rows ? int(max(int64_t(-1), s.before + r / group)) : -1;
            }
        }
        // Units that every row sees whole: up to `sees_all`, from `window_all` on.
        const int last_row = min(row0 + kRows, rows) - 1;
        const int sees_all = int(max(int64_t(0), min(s.before + row0 / group + 1, int64_t(s.length))) / kUnit);
        const int window_all = a.window > 0 ? int(min(max(int64_t(0), s.before + last_row / group - a.window + 1) + kUnit - 1, int64_t(0x7fffffff)) / kUnit) : 0;

        uint32_t base[kGroups];  // the middle, as codes are before it is taken off
        float middle[kGroups];
#pragma unroll
        for (int b = 0; b < kGroups; ++b) base[b] = 0x64086408u, middle[b] = kMiddle;
        float acc[NT][kGroups][4][4], least[NT][kGroups][2];
        float top[NT][2], against[NT][2], sum[NT][2];  // maxima of scores before `to_log2`
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int b = 0; b < kGroups; ++b) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int m = 0; m < 4; ++m) acc[j][b][m][i] = 0.f;
                }
                least[j][b][0] = least[j][b][1] = 0.f;
            }
            top[j][0] = top[j][1] = kNone;
            sum[j][0] = sum[j][1] = 0.f;
            against[j][0] = against[j][1] = C::kNarrow ? -kNone : 0.f;
        }
        int next_ahead = 0;
        const int next_mine = units_of(next);
#pragma unroll 1
        for (int i = 0; i < mine && !gave_up; ++i) {
            if (!__all_sync(~0u, tc::bar_wait_or_look(&bars[warp][stage], phase, &abort_flag, a.wait_clocks))) {
                gave_up = true;
                break;
            }
            missing &= ~(1u << (kArmed + stage));
            const uint8_t *const unit = ring + stage * Shape::kStage;
            const int index = s.unit + warp + i * kWarps;
            const uint32_t none = missing >> 2 * stage & 3;
            if (C::kNarrow && i == 0) {
                // The code that sums over tokens are about: the whole number nearest to zero's in this warp's first tokens.
                // About 8, with values whose extremes are far from symmetric, sums that the tensor cores cut off were 5e-3 of
                // the outputs' norm off at 14000 tokens a warp (bf16: 2.9e-3, of which its own roundings are 2.4e-3; there it
                // costs 357 -> 384 us with 256 requests, here 385 -> 403).
                float steps[kGroups] = {}, lows[kGroups] = {};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t pairs[kGroups];
                    load_words(unit + (e >> 1) * Tile::kBytes + Tile::kValuePairs + (g + 8 * (e & 1)) * kGroups * 4, pairs);
                    const int p = index * kUnit + 8 * e + (g >> 1) + 4 * (g & 1);
                    if (p >= here.seen_from && p < s.length && !(none >> (e >> 1) & 1)) {
#pragma unroll
                        for (int b = 0; b < kGroups; ++b) steps[b] += pair_scale(pairs[b]), lows[b] += pair_min(pairs[b]);
                    }
                }
#pragma unroll
                for (int b = 0; b < kGroups; ++b) {
                    const float at = 15.f * __saturatef(-lows[b] * reciprocal_approx(15.f * steps[b]));
                    const uint32_t code = (__reduce_add_sync(~0u, steps[b] > 0.f ? __float2uint_rn(at) : 8u) + 16) / 32;  // the lanes' mean
                    base[b] = 0x64006400u + code * 0x10001u;
                    middle[b] = float(code);
                }
            }
            // Scores of tokens (rows g, g + 8 of each tile) x query rows (2 t, 2 t + 1).
            float z[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t *const tile = unit + h * Tile::kBytes;
#pragma unroll
                for (int j = 0; j < NT; ++j) z[h][j][0] = z[h][j][1] = z[h][j][2] = z[h][j][3] = 0.f;
                uint32_t key_pairs[2][kGroups];
                load_words(tile + Tile::kKeyPairs + g * kGroups * 4, key_pairs[0]);
                load_words(tile + Tile::kKeyPairs + (g + 8) * kGroups * 4, key_pairs[1]);
#pragma unroll
                for (int block = 0; block < kGroups / Tile::kBlockGroups; ++block) {
                    uint32_t lo[2 * Tile::kBlockGroups], hi[2 * Tile::kBlockGroups];
                    const uint8_t *from = tile + block * kTile * Tile::kBlockRow + t * 8 * Tile::kBlockGroups;
                    load_words(from + g * Tile::kBlockRow, lo);
                    load_words(from + (g + 8) * Tile::kBlockRow, hi);
#pragma unroll
                    for (int half = 0; half < Tile::kBlockGroups; ++half) {
                        const int b = block * Tile::kBlockGroups + half;
                        float d[NT][4];
#pragma unroll
                        for (int j = 0; j < NT; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const uint32_t x = lo[2 * half + w], y = hi[2 * half + w];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t a0 = C::pair(x >> (8 * k)), a1 = C::pair(y >> (8 * k));
                                const uint32_t a2 = C::pair(x >> (8 * k + 4)), a3 = C::pair(y >> (8 * k + 4));
#pragma unroll
                                for (int j = 0; j < NT; ++j) C::mma(d[j], a0, a1, a2, a3, q[j][b][4 * w + 2 * k], q[j][b][4 * w + 2 * k + 1]);
                            }
                        }
                        const float s0 = pair_scale(key_pairs[0][b]), s1 = pair_scale(key_pairs[1][b]);
                        const float m0 = pair_min(key_pairs[0][b]) - C::kHeld * s0, m1 = pair_min(key_pairs[1][b]) - C::kHeld * s1;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            z[h][j][0] += s0 * d[j][0] + m0 * q_sum[j][b][0];
                            z[h][j][1] += s0 * d[j][1] + m0 * q_sum[j][b][1];
                            z[h][j][2] += s1 * d[j][2] + m1 * q_sum[j][b][0];
                            z[h][j][3] += s1 * d[j][3] + m1 * q_sum[j][b][1];
                        }
                    }
                }
            }
            uint32_t hidden = 0;  // bits of z
            if (index >= sees_all || index < window_all || none) {
                // Row r of a tile is token r / 2 + 4 (r % 2) of its half.
                const int token = index * kUnit + (g >> 1) + 4 * (g & 1);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) {
                            const int p = token + h * kTile + (i4 & 2) * 4, own = place[j][i4 & 1];
                            if (p > own || p >= s.length || (a.window > 0 && p <= own - a.window) || (none >> h & 1)) {
                                hidden |= 1u << (4 * (h * NT + j) + i4);
                                z[h][j][i4] = -INFINITY;
                            }
                        }
            }
            float most[NT][2];
            bool grows = false;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    most[j][e] = fmaxf(fmaxf(z[0][j][e], z[0][j][2 + e]), fmaxf(z[1][j][e], z[1][j][2 + e]));
                    if constexpr (C::kNarrow) grows = grows || fmaf(most[j][e], to_log2, against[j][e]) > C::kMostPower;
                    else grows = grows || most[j][e] > top[j][e] + lag;
                }
            auto rescale = [&](int j, int e, float factor) {
                sum[j][e] *= factor;
#pragma unroll
                for (int b = 0; b < kGroups; ++b) {
                    least[j][b][e] *= factor;
#pragma unroll
                    for (int m = 0; m < 4; ++m) acc[j][b][m][e] *= factor, acc[j][b][m][2 + e] *= factor;
                }
            };
            // The maxima that weights are taken against may lag behind by 2^kLag: they move seldom.
            if (__any_sync(~0u, grows)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = most[j][e];
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                        float factor;
                        if constexpr (C::kNarrow) {
                            const float now = fminf(against[j][e], C::kLag - x * to_log2);
                            factor = exp2_approx(now - against[j][e]);
                            against[j][e] = now;
                        } else {
                            x = fmaxf(x, top[j][e]);
                            factor = exp2_approx((top[j][e] - x) * to_log2);
                            top[j][e] = x;
                            against[j][e] = x == kNone ? 0.f : -x * to_log2;  // (a row that has seen nothing yet)
                        }
                        rescale(j, e, factor);
                    }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        z[h][j][i4] = exp2_approx(fmaf(z[h][j][i4], to_log2, against[j][i4 & 1]));
                        sum[j][i4 & 1] += z[h][j][i4];
                    }
            if constexpr (C::kNarrow) {
                float scale[2][2];  // largest of a token's groups
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t pairs[kGroups];
                        load_words(unit + h * Tile::kBytes + Tile::kValuePairs + (g + 8 * i) * kGroups * 4, pairs);
                        scale[h][i] = pair_scale(pairs[0]);
#pragma unroll
                        for (int b = 1; b < kGroups; ++b) scale[h][i] = fmaxf(scale[h][i], pair_scale(pairs[b]));
                    }
                // NaN aside, which a hidden token's may be too: its weight is 0.
                auto largest = [&](int j, int e) {
                    return fmaxf(fmaxf(z[0][j][e] * scale[0][0], z[0][j][2 + e] * scale[0][1]),
                                 fmaxf(z[1][j][e] * scale[1][0], z[1][j][2 + e] * scale[1][1]));
                };
                bool over = false;
#pragma unroll
                for (int j = 0; j < NT; ++j) over = over || fmaxf(largest(j, 0), largest(j, 1)) > C::kMostWeight;
                if (__any_sync(~0u, over)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = largest(j, e);
                            x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                            const int less = x > C::kMostWeight ? int(__float_as_uint(x) >> 23) - 127 - 8 : 0;
                            const float factor = __uint_as_float(uint32_t(127 - less) << 23);
                            against[j][e] -= float(less);
                            rescale(j, e, factor);
#pragma unroll
                            for (int h = 0; h < 2; ++h) z[h][j][e] *= factor, z[h][j][2 + e] *= factor;
                        }
                }
            }
            // Values: rows are channels (x: even ones, y: odd ones), columns query rows.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t *const tile = unit + h * Tile::kBytes;
                uint32_t value_pairs[2][kGroups], word[4][kGroups];
                load_words(tile + Tile::kValuePairs + g * kGroups * 4, value_pairs[0]);
                load_words(tile + Tile::kValuePairs + (g + 8) * kGroups * 4, value_pairs[1]);
                const uint8_t *from = tile + Tile::kValues + (kGroups * g >> 3) * kTile * 32 + (kGroups * g & 7) * 4 + t * 32;
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) load_words(from + i4 * 4 * 32, word[i4]);
#pragma unroll
                for (int b = 0; b < kGroups; ++b) {
                    // A weight p s is rounded before it meets a code, so the rest of the value has to go by the rounded weight
                    // too, or what is lost is not p v's but that of two parts that cancel: with weights nearly alike, whose
                    // roundings are then alike, that was up to 12 % of the outputs' norm (20000 tokens).  With zero's code k (0
                    // to 15, the nearest where zero is outside): p v = p s (c - k) + p (m + k s), the second part 0 or, where
                    // all of a group's values have one sign, the smallest of them.  (256 requests 338 -> 357 us.)
                    // Here 8 - k and m + k s; any k in that range gives the same sum but for roundings.
                    auto zero_of = [&](float step, float low, float &below, float &rest) {
                        const float range = 15.f * step, at = __saturatef(-low * reciprocal_approx(range));
                        below = fmaf(at, -15.f, middle[b]);
                        rest = fmaf(at, range, low);
                    };
                    const float s0 = pair_scale(value_pairs[0][b]), s1 = pair_scale(value_pairs[1][b]);
                    float below0, below1, rest0, rest1;
                    zero_of(s0, pair_min(value_pairs[0][b]), below0, rest0);
                    zero_of(s1, pair_min(value_pairs[1][b]), below1, rest1);
                    uint32_t w0[NT], w1[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float u[4] = {z[h][j][0] * s0, z[h][j][1] * s0, z[h][j][2] * s1, z[h][j][3] * s1};
                        if (hidden) {  // a hidden token's scale and minimum may be anything
#pragma unroll
                            for (int i4 = 0; i4 < 4; ++i4)
                                if (hidden >> (4 * (h * NT + j) + i4) & 1) u[i4] = 0.f;
                        }
                        w0[j] = C::pack(u[0], u[1]);
                        w1[j] = C::pack(u[2], u[3]);
                        const float2 r0 = C::unpack(w0[j]), r1 = C::unpack(w1[j]);
                        if (hidden) {
                            const float v[4] = {fmaf(r0.x, below0, z[h][j][0] * rest0), fmaf(r0.y, below0, z[h][j][1] * rest0),
                                                fmaf(r1.x, below1, z[h][j][2] * rest1), fmaf(r1.y, below1, z[h][j][3] * rest1)};
#pragma unroll
                            for (int i4 = 0; i4 < 4; ++i4)
                                if (!(hidden >> (4 * (h * NT + j) + i4) & 1)) least[j][b][i4 & 1] += v[i4];
                        } else {
                            least[j][b][0] = fmaf(r1.x, below1, fmaf(z[h][j][2], rest1, fmaf(r0.x, below0, fmaf(z[h][j][0], rest0, least[j][b][0]))));
                            least[j][b][1] = fmaf(r1.y, below1, fmaf(z[h][j][3], rest1, fmaf(r0.y, below0, fmaf(z[h][j][1], rest0, least[j][b][1]))));
                        }
                        w0[j] = transpose8(w0[j]);
                        w1[j] = transpose8(w1[j]);
                    }
                    const uint32_t x0 = __byte_perm(word[0][b], word[1][b], 0x5410), y0 = __byte_perm(word[0][b], word[1][b], 0x7632);
                    const uint32_t x1 = __byte_perm(word[2][b], word[3][b], 0x5410), y1 = __byte_perm(word[2][b], word[3][b], 0x7632);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const uint32_t a0 = C::centred(x0 >> (4 * m), base[b]), a1 = C::centred(y0 >> (4 * m), base[b]);
                        const uint32_t a2 = C::centred(x1 >> (4 * m), base[b]), a3 = C::centred(y1 >> (4 * m), base[b]);
#pragma unroll
                        for (int j = 0; j < NT; ++j) C::mma(acc[j][b][m], a0, a1, a2, a3, w0[j], w1[j]);
                    }
                }
            }
            __syncwarp();
            stage = stage + 1 == kStages ? 0 : stage + 1;
            phase ^= stage == 0;
            if (ahead < mine) request(here, ahead++);
            else if (next_ahead < next_mine) request(next, next_ahead++);
        }
        ahead = next_ahead;

        // The warps' sums, to shared memory, then to the output or a part.
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = j * 8 + 2 * t + e;
                float total = sum[j][e];
#pragma unroll
                for (int i = 4; i < 32; i *= 2) total += __shfl_xor_sync(~0u, total, i);
                if (g == 0) row_max[warp][row] = gave_up ? NAN : !C::kNarrow && top[j][e] == kNone ? kNone : -against[j][e], row_sum[warp][row] = total;
#pragma unroll
                for (int b = 0; b < kGroups; ++b) {
                    float low_part = least[j][b][e];
#pragma unroll
                    for (int i = 4; i < 32; i *= 2) low_part += __shfl_xor_sync(~0u, low_part, i);
                    float *to = merge + (warp * kRows + row) * Shape::kMergeRow + b * kGroup + 8 * g;
#pragma unroll
                    for (int m = 0; m < 4; m += 2)
                        *reinterpret_cast<float4 *>(to + 2 * m) =
                            make_float4(acc[j][b][m][e] + low_part, acc[j][b][m][2 + e] + low_part, acc[j][b][m + 1][e] + low_part,
                                        acc[j][b][m + 1][2 + e] + low_part);
                }
            }
        __syncthreads();
        const int warps = min(s.count, kWarps);  // that had units
        const int64_t slot = 2 * blockIdx.x + (number == 0 ? 0 : 1);
        float *part = reinterpret_cast<float *>(a.workspace) + slot * Shape::kPart;
        for (int i = threadIdx.x; i < kRows * D / 4; i += kAttnThreads) {
            const int row = i / (D / 4), c = i % (D / 4) * 4;
            float most = kNone;
            bool bad = false;
            for (int w = 0; w < warps; ++w) {
                most = fmaxf(most, row_max[w][row]);
                bad = bad || row_max[w][row] != row_max[w][row];
            }
            if (bad) most = NAN;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float weight = 0.f;
            for (int w = 0; w < warps; ++w) {
                const float factor = exp2_approx(row_max[w][row] - most);
                const float4 y = *reinterpret_cast<const float4 *>(merge + (w * kRows + row) * Shape::kMergeRow + c);
                x.x += factor * y.x, x.y += factor * y.y, x.z += factor * y.z, x.w += factor * y.w;
                weight += factor * row_sum[w][row];
            }
            if (s.whole) {
                if (row0 + row < rows) {
                    const float per = weight == 0.f ? 0.f : 1.f / weight;
                    const int token = (row0 + row) / group, head = s.head * group + row0 + row - token * group;
                    T *out = static_cast<T *>(a.out) + ((int64_t(s.first) + token) * a.q_heads + head) * D + c;
                    *reinterpret_cast<uint2 *>(out) = make_uint2(C::pack(x.x * per, x.y * per), C::pack(x.z * per, x.w * per));
                }
            } else {
                *reinterpret_cast<float4 *>(part + row * D + c) = x;
                if (c == 0) part[kRows * D + row] = most, part[kRows * D + kRows + row] = weight;
            }
        }
        __syncthreads();
    }
    if (gave_up) {  // the copies still on their way end before the CTA does
        if (lane == 0) flag(a.status, SQ_STATUS_TIMEOUT);
        int alone = 0;
        for (int i = 0; i < kStages; ++i)
            if (missing >> (kArmed + i) & 1) tc::bar_wait(&bars[warp][i], i < stage ? phase ^ 1 : phase, &alone, tc::kWaitClocks);
    }
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    // Beside prompts it started when their last CTAs had: what comes after it in the stream waits for them too.
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

// Joins the parts of items that several CTAs had: CTAs (c, y), c that in whose span an item ends, take a
// quarter of its sums each.
constexpr int kJoins = 4;

template <class T, int D, int NT>
__global__ void __launch_bounds__(kAttnThreads) join_kernel(sq_kv_attention_args a, int most_rows) {
    using Shape = RowsShape<D, NT>;
    using C = Codes<T>;
    constexpr int kRows = Shape::kRows, kMine = kRows * D / 4 / kJoins, kSplit = kAttnThreads / kMine;  // accesses of four; threads to each
    extern __shared__ float factors[];  // [parts][rows]
    __shared__ float weights[kRows];
    __shared__ float4 sums[kAttnThreads];
    const Span span = span_of<kRows>(a, most_rows, false);
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (span.begin >= span.end) return;
    const Sequence seq = sequence<kRows>(a, most_rows, span.sequence, false);
    const int per_item = kItemUnits + seq.units, done = int(span.offset - quotient(span.offset, per_item) * per_item);  // of the item, before this span
    if (done <= kItemUnits || per_item - done > span.end - span.begin) return;
    // The first part is that of the CTA with the item's first unit: its only segment where its span begins in the item.
    const int item = int(quotient(span.offset, per_item));
    const int64_t start = span.begin - done, cta0 = quotient(start + kItemUnits, span.per);
    const int head = item / seq.blocks, block = item % seq.blocks, parts = int(blockIdx.x - cta0) + 1;
    const float *workspace = static_cast<const float *>(a.workspace);
    auto part = [&](int i) {
        const int64_t slot = 2 * (cta0 + i) + (i == 0 && cta0 * span.per < start ? 1 : 0);
        return workspace + slot * Shape::kPart;
    };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int row = warp; row < kRows; row += kWarps) {
        float most = kNone;
        bool bad = false;
        for (int i = lane; i < parts; i += 32) {
            const float x = part(i)[kRows * D + row];
            factors[i * kRows + row] = x;
            most = fmaxf(most, x);
            bad = bad || x != x;
        }
#pragma unroll
        for (int i = 1; i < 32; i *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, i));
        if (__any_sync(~0u, bad)) most = NAN;
        float weight = 0.f;
        for (int i = lane; i < parts; i += 32) {
            const float f = exp2_approx(factors[i * kRows + row] - most);
            factors[i * kRows + row] = f;
            weight += f * part(i)[kRows * D + kRows + row];
        }
#pragma unroll
        for (int i = 1; i < 32; i *= 2) weight += __shfl_xor_sync(~0u, weight, i);
        if (lane == 0) weights[row] = weight;
    }
    __syncthreads();
    const int i = blockIdx.y * kMine + threadIdx.x % kMine, row = i / (D / 4), c = i % (D / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = threadIdx.x / kMine; p < parts; p += kSplit) {
        const float f = factors[p * kRows + row];
        const float4 y = *reinterpret_cast<const float4 *>(part(p) + row * D + c);
        x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
    }
    sums[threadIdx.x] = x;
    __syncthreads();
    const int row0 = block * kRows, rows = seq.count * (a.q_heads / a.heads);
    if (threadIdx.x >= kMine || row0 + row >= rows) return;
#pragma unroll
    for (int k = 1; k < kSplit; ++k) {
        const float4 y = sums[threadIdx.x + k * kMine];
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    const float per = weights[row] == 0.f ? 0.f : 1.f / weights[row];
    T *out = output_row<T>(a, seq, head, row0 + row) + c;
    *reinterpret_cast<uint2 *>(out) = make_uint2(C::pack(x.x * per, x.y * per), C::pack(x.z * per, x.w * per));
}

template <class T, int D, int NT>
cudaError_t launch_rows(const sq_kv_attention_args &a, int most_rows, bool beside, cudaStream_t s) {
    using Shape = RowsShape<D, NT>;
    const int sms = sms_of(s);
    if (sms < 1) return cudaErrorInvalidDevice;
    const int resident = NT == 1 && D <= 128 ? 2 : 1;
    const unsigned grid = unsigned(sms * resident < kMostCtas ? sms * resident : kMostCtas);
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = allow_shared(rows_kernel<T, D, NT>, Shape::kShared, devices);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = Shape::kShared;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = beside ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, rows_kernel<T, D, NT>, a, most_rows);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(grid, kJoins);
    cfg.dynamicSmemBytes = size_t(grid) * Shape::kRows * sizeof(float);
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<T, D, NT>, a, most_rows);
}

// Blocks of 16 rows where sequences have more than 8 (heads of 256 channels: their sums leave no room).
bool wide_rows(int tokens, int seqs, int q_heads, int heads, int dim) {
    return dim < 256 && int64_t(tokens) * (q_heads / heads) > int64_t(seqs) * 8;
}

template <class T>
cudaError_t launch_rows(const sq_kv_attention_args &a, int most_rows, bool beside, cudaStream_t s) {
    const bool wide = wide_rows(a.tokens, a.num_seqs, a.q_heads, a.heads, a.dim);
    switch (a.dim) {
        case 64: return wide ? launch_rows<T, 64, 2>(a, most_rows, beside, s) : launch_rows<T, 64, 1>(a, most_rows, beside, s);
        case 128: return wide ? launch_rows<T, 128, 2>(a, most_rows, beside, s) : launch_rows<T, 128, 1>(a, most_rows, beside, s);
        default: return launch_rows<T, 256, 1>(a, most_rows, beside, s);
    }
}

// Sequences of up to kFewRows rows (new tokens times query heads of a kv head) go through rows_kernel, those
// of more through the prompts' kernel, each decided on the device: a batch may have both.  The few rows are a
// programmatic dependent of the prompts, whose outputs they do not touch: they fill the SMs that the prompts'
// last CTAs leave (8 ragged prompts, two of them short: 318 us one after the other).
cudaError_t launch_attention(const sq_kv_attention_args &a, cudaStream_t s) {
    const int group = a.q_heads / a.heads;
    const bool prompts = a.cu_seqlens && group <= 128 && int64_t(a.tokens) * group > kFewRows;
    const int most_rows = prompts ? kFewRows : 0x7fffffff;
    if (prompts) {
        const cudaError_t e = launch_prompt_attention(a, kFewRows, s);
        if (e != cudaSuccess) return e;
    }
    return a.dtype == SQ_BF16 ? launch_rows<__nv_bfloat16>(a, most_rows, prompts, s) : launch_rows<__half>(a, most_rows, prompts, s);
}

}  // namespace
}  // namespace sq

extern "C" int64_t sq_kv_attention_workspace_bytes(int32_t tokens, int32_t num_seqs, int32_t q_heads, int32_t heads, int32_t dim) {
    if (tokens < 0 || num_seqs < 0 || heads < 1 || q_heads < 1 || (dim != 64 && dim != 128 && dim != 256)) return -1;
    if (tokens == 0 || num_seqs == 0) return 0;
    const int64_t rows = sq::wide_rows(tokens, num_seqs, q_heads, heads, dim) ? 16 : 8;
    return 2 * sq::kMostCtas * (rows * dim + 2 * rows) * int64_t(sizeof(float));
}

extern "C" int32_t sq_kv_attention(const sq_kv_attention_args *args, sq_stream_t stream) {
    using namespace sq;
    if (!args) return SQ_ERR_ARGUMENT;
    sq_kv_attention_args a = *args;
    if (a.tokens < 0 || a.num_seqs < 0 || a.table_width < 0 || a.num_pages < 0 || a.heads < 1 || a.q_heads < 1 || a.window < 0)
        return SQ_ERR_ARGUMENT;
    if (a.dtype < SQ_F32 || a.dtype > SQ_F16 || !(a.scale > 0.f) || !(a.scale < INFINITY)) return SQ_ERR_ARGUMENT;
    if (a.dtype == SQ_F32 || (a.dim != 64 && a.dim != 128 && a.dim != 256)) return SQ_ERR_UNSUPPORTED;
    if (a.page_size < kTile || a.page_size % kTile || a.table_stride < 0 || a.q_heads % a.heads) return SQ_ERR_SHAPE;
    if (a.q_stride < 0 || a.q_head_stride < 0 || a.q_stride % 8 || a.q_head_stride % 8) return SQ_ERR_SHAPE;
    if (!aligned16(a.q) || !aligned16(a.out) || !aligned16(a.data) || !aligned16(a.workspace)) return SQ_ERR_SHAPE;
    if (a.heads > 4096 || a.q_heads > 65536 || a.page_size > 65536 || a.tokens > kMostTokens || a.num_seqs > (1 << 30))
        return SQ_ERR_UNSUPPORTED;
    if (int64_t(a.tokens) * (a.q_heads / a.heads) > kMostTokens) return SQ_ERR_UNSUPPORTED;  // rows of a kv head
    if (int64_t(a.table_width) * a.page_size > kMostTokens) return SQ_ERR_UNSUPPORTED;  // positions are ints
    if (!a.cu_seqlens && a.tokens != a.num_seqs) return SQ_ERR_ARGUMENT;
    if (a.tokens == 0 || a.num_seqs == 0) return SQ_OK;
    if (!a.q || !a.out || !a.lengths || (a.table_width && !a.page_table) || (a.num_pages && !a.data)) return SQ_ERR_ARGUMENT;
    if (!a.workspace || a.workspace_bytes < sq_kv_attention_workspace_bytes(a.tokens, a.num_seqs, a.q_heads, a.heads, a.dim))
        return SQ_ERR_CAPACITY;
    if (a.wait_clocks == 0) a.wait_clocks = tc::kWaitClocks;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return launch_attention(a, s) == cudaSuccess ? SQ_OK : SQ_ERR_CUDA;
}
