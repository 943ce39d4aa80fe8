// Attention of prompts over the paged 4-bit cache, on tcgen05 (sq_attention.cu has few rows).
//
// A CTA takes 256 query rows of one kv head, (token, query head) pairs, in two tiles of
// 128 (heads of 256 channels: one tile, as its sums fill the tensor memory), and walks
// the keys in blocks of 128 (64).  Per block:
//   four warps (eight) write out the codes as 16-bit keys and values in shared memory,
//   one thread issues S = Q K^T and O += P V, S, P and O in tensor memory,
//   four warps a tile, a thread to a row, turn S into P, which overwrites it.
// While a tile's S becomes P, the other tile's products run (one tile: the next block's S).
// Scores take keys as they are held: s (c - 8) has 3 + 8 significant bits and so is an f16,
// and the rest of a group, m + 8 s, meets the sum of the query's channels in one more step
// of K (the sum's f16 and its remainder, each by m and by 8 s).  Queries are f16 with each
// row's largest value near 2^8, keys over 16.  Values m + s c and weights are rounded to f16
// too, whatever the cache's type, values times a power of two that brings the largest of
// the item's keys near 2^14, which a scan of their scales and minima finds first (bf16
// values and weights were half as exact: 2.6e-3 of an output's norm, of which 1.7e-3 are
// its own rounding).
// Row maxima may lag by 2^8, so sums in tensor memory are seldom rescaled.
#include "sq_kv.cuh"
#include "sq_rows.cuh"
#include "sq_tc.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kPromptThreads = 13 * 32;
constexpr float kKeyDivisor = 16.f;
constexpr float kPromptLag = 8.f;

template <int D>
struct PromptShape {
    using Tile = KvTile<D>;
    static constexpr int kTiles = D == 256 ? 1 : 2;             // of 128 rows
    static constexpr int kKeys = D == 256 ? 64 : 128;           // of a block
    static constexpr int kSoftmaxWarps = 4 * kTiles, kUnpackThreads = 32 * (12 - kSoftmaxWarps);
    static constexpr int kQueryBytes = 128 * D * 2, kKeyBytes = kKeys * D * 2;
    static constexpr int kMoreQuery = 128 * 32, kMoreKey = kKeys * 32;  // the last step of K: 16 values a row
    static constexpr int kShared = kTiles * (kQueryBytes + kMoreQuery) + 4 * kKeyBytes + 2 * kMoreKey + 1024;
    static constexpr int kColumnsO = 2 * kKeys;                 // S, P: [0, 2 kKeys)
    static constexpr int kPieces = kKeys * D / 32 / kUnpackThreads;  // 16-byte pieces of a block's keys for a thread
    static_assert(kColumnsO + kTiles * D <= 512 && kPieces * kUnpackThreads * 32 == kKeys * D, "");
};

struct PromptBars {
    uint64_t query, keys[2], keys_free[2], values[2], values_free[2], scores[2], weights[2], sums[2], end;
};

// Codes of 8 channels as f16 pairs (c - 8) s, or as pairs c s + m.
__device__ __forceinline__ uint4 unpack_middle(uint32_t w, __half2 s) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u, base = 0x64086408u;  // 1024 + c less 1032
        const __half2 v = __hmul2(__hsub2(reinterpret_cast<const __half2 &>(x), reinterpret_cast<const __half2 &>(base)), s);
        r[i] = reinterpret_cast<const uint32_t &>(v);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint4 unpack_f16(uint32_t w, __half2 s, __half2 m) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u, base = 0x64006400u;
        const __half2 c = __hsub2(reinterpret_cast<const __half2 &>(x), reinterpret_cast<const __half2 &>(base));
        const __half2 v = __hfma2(c, s, m);
        r[i] = reinterpret_cast<const uint32_t &>(v);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ float low_bf16(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_bf16(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) { return make_float2(low_bf16(x), high_bf16(x)); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) { return __half22float2(reinterpret_cast<const __half2 &>(x)); }

// Item of a CTA.
struct PromptItem {
    int first, count;    // the sequence's new tokens
    int token, rows;     // first token of the item in it, rows (token, query head)
    int length, head;
    int64_t before;      // position of the sequence's first new token
    int start, blocks;   // first key, a multiple of 16; blocks of keys
    const int32_t *table;
};

// Byte offset of a tile of 16 keys that begins at `key`, or -1.
template <int D>
__device__ __forceinline__ int64_t prompt_tile(const sq_kv_attention_args &a, const PromptItem &item, int key) {
    if (key >= item.length) return -1;
    const int page = item.table[key / a.page_size];
    if (page <= 0) return -1;
    if (page >= a.num_pages) {
        flag(a.status, SQ_STATUS_SLOT_RANGE);
        return -1;
    }
    return ((int64_t(page) * a.heads + item.head) * (a.page_size / kTile) + key % a.page_size / kTile) * KvTile<D>::kBytes;
}

template <class T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_kernel(sq_kv_attention_args a, int tokens_per_item, unsigned strips, int few_rows) {
    using Shape = PromptShape<D>;
    using Tile = KvTile<D>;
    constexpr int kTiles = Shape::kTiles, kKeys = Shape::kKeys, kGroups = Tile::kGroups;
    extern __shared__ uint8_t raw[];
    __shared__ PromptBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, bad_values;
    __shared__ unsigned most_value;
    __shared__ volatile int holes[4];  // block + 1 of the last one with tiles to leave out, by block modulo 4
    uint8_t *const queries = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t *const keys = queries + kTiles * Shape::kQueryBytes, *const values = keys + 2 * Shape::kKeyBytes;
    uint8_t *const more_queries = values + 2 * Shape::kKeyBytes, *const more_keys = more_queries + kTiles * Shape::kMoreQuery;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.q_heads / a.heads;

    // Later strips, which see more keys, first.
    PromptItem item;
    {
        const unsigned strip = strips - 1 - blockIdx.x / a.heads;
        item.head = int(blockIdx.x % a.heads);
        const int n = sequence_of(a.cu_seqlens, a.num_seqs, a.tokens, tokens_per_item, strip);
        const int2 r = sequence_range(a.cu_seqlens, n, a.tokens);
        item.first = r.x;
        item.count = r.y - r.x;
        const int64_t token = (int64_t(strip) - (int64_t(r.x) / tokens_per_item + n)) * tokens_per_item;
        if (token < 0 || token >= item.count || int64_t(item.count) * group <= few_rows) return;
        item.token = int(token);
        const int tokens = min(tokens_per_item, item.count - item.token);
        item.rows = tokens * group;
        const int64_t length = a.lengths[n], most = int64_t(a.table_width) * a.page_size;
        if (length > most && threadIdx.x == 0) flag(a.status, SQ_STATUS_SLOT_RANGE);
        item.length = int(max(int64_t(0), min(length, most)));
        item.before = length - item.count;
        item.table = a.page_table + n * a.table_stride;
        const int64_t low = item.before + item.token, high = min(low + tokens, int64_t(item.length));
        item.start = a.window > 0 ? int(min(max(int64_t(0), low - a.window + 1), int64_t(item.length)) & ~int64_t(kTile - 1)) : 0;
        item.blocks = int(max(int64_t(0), high - item.start + kKeys - 1) / kKeys);
    }
    const int live = item.rows > 128 ? kTiles : 1;  // tiles of rows

    if (warp == 12) {
        tc::tmem_alloc(&tmem_slot, 512);
        if (lane == 0) {
            tc::bar_init(&bars.query, 4 * live);
            for (int i = 0; i < 2; ++i) {
                tc::bar_init(&bars.keys[i], Shape::kUnpackThreads / 32);
                tc::bar_init(&bars.values[i], Shape::kUnpackThreads / 32);
                tc::bar_init(&bars.keys_free[i], 1);
                tc::bar_init(&bars.values_free[i], 1);
                tc::bar_init(&bars.scores[i], 1);
                tc::bar_init(&bars.weights[i], 4);
                tc::bar_init(&bars.sums[i], 1);
            }
            tc::bar_init(&bars.end, 1);
            tc::bar_init_fence();
            abort_flag = 0;
            bad_values = 0;
            most_value = 0;
            for (int i = 0; i < 4; ++i) holes[i] = 0;
        }
        __syncwarp();
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_slot;

    // Largest |m| + 15 s of the item's values.
    {
        constexpr int kEach = D / 16;  // accesses of four pairs a tile
        const int64_t end = min(int64_t(item.start) + int64_t(item.blocks) * kKeys, int64_t(item.length));
        float most = 0.f;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < (end - item.start + kTile - 1) / kTile * kEach; i += kPromptThreads) {
            const int key = item.start + int(i / kEach) * kTile, first = int(i % kEach) * 4;
            const int64_t at = prompt_tile<D>(a, item, key);
            if (at < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4 *>(a.data + at + Tile::kValuePairs + first * 4);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = (first + e) / kGroups, token = (row & 8) | ((row & 1) << 2) | ((row >> 1) & 3);
                if (key + token < item.length) most = fmaxf(most, fabsf(high_bf16(w[e])) + 15.f * low_bf16(w[e]));
            }
        }
#pragma unroll
        for (int i = 1; i < 32; i *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, i));
        if (lane == 0) atomicMax(&most_value, __float_as_uint(fminf(most, 3e38f)));
        __syncthreads();
    }
    const int value_shift = most_value == 0 ? 0 : max(-100, min(100, 14 - (int(most_value >> 23) - 127)));
    const float value_factor = __uint_as_float(uint32_t(127 + value_shift) << 23);
    auto wait_alone = [&](uint64_t *bar, uint32_t parity) { return tc::bar_wait(bar, parity, &abort_flag, tc::kWaitClocks); };
    auto wait = [&](uint64_t *bar, uint32_t parity) { return bool(__all_sync(~0u, wait_alone(bar, parity))); };  // of a whole warp

    float top = -INFINITY;  // of a row
    float2 sum = make_float2(0.f, 0.f);  // of its weights, in two parts
    if (warp < Shape::kSoftmaxWarps) {
        const int tile = warp >> 2, row = threadIdx.x & 127, index = tile * 128 + row;
        if (tile < live) {
            const bool mine = index < item.rows;
            const int token = item.token + (mine ? index / group : 0);
            // The row's query, times a power of two that brings its largest value to [2^8, 2^9).
            const T *q = static_cast<const T *>(a.q) + int64_t(item.first + token) * a.q_stride +
                         (item.head * group + (mine ? index % group : 0)) * a.q_head_stride;
            float most = 0.f;
#pragma unroll 8
            for (int i = 0; i < D / 8; ++i) {
                const uint4 x = reinterpret_cast<const uint4 *>(q)[i];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = unpack2<T>(w[e]);
                    most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            const int exponent = int(__float_as_uint(most) >> 23);
            const int shift = most == 0.f || exponent == 255 ? 0 : min(8 - (exponent - 127), 126);
            const float factor = __uint_as_float(uint32_t(127 + shift) << 23);
            uint8_t *const to = queries + tile * Shape::kQueryBytes + row * 128;
            uint32_t more[8] = {};  // for each group its sum's f16 and remainder, twice
            float group_sum = 0.f;
#pragma unroll 8
            for (int i = 0; i < D / 8; ++i) {
                const uint4 x = reinterpret_cast<const uint4 *>(q)[i];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = unpack2<T>(w[e]);
                    r[e] = mine ? pack2<__half>(v.x * factor, v.y * factor) : 0;
                    const float2 rounded = unpack2<__half>(r[e]);
                    group_sum += rounded.x + rounded.y;
                }
                if ((i & 7) == 7) {
                    const float high = __half2float(__float2half_rn(group_sum));
                    const uint32_t both = pack2<__half>(high, group_sum - high);
#pragma unroll
                    for (int b = 0; b < kGroups; ++b)
                        if (b == i / 8) more[2 * b] = more[2 * b + 1] = both;
                    group_sum = 0.f;
                }
                *reinterpret_cast<uint4 *>(to + (i >> 3) * 16384 + (((i & 7) ^ (row & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
            }
            uint8_t *const more_to = more_queries + tile * Shape::kMoreQuery + row * 16;
            *reinterpret_cast<uint4 *>(more_to) = make_uint4(more[0], more[1], more[2], more[3]);
            *reinterpret_cast<uint4 *>(more_to + 128 * 16) = make_uint4(more[4], more[5], more[6], more[7]);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::bar_arrive(&bars.query);
            const float to_log2 = a.scale * kLog2e * kKeyDivisor / factor;
            const int64_t last = mine ? min(item.before + token, int64_t(item.length) - 1) : -1;
            const uint32_t lanes = uint32_t(warp & 3) << 21;
            const uint32_t sums = tmem + lanes + Shape::kColumnsO + tile * D;
            bool ok = true;
            for (int j = 0; j < item.blocks && ok; ++j) {
                const int buffer = kTiles == 2 ? tile : j & 1;
                const uint32_t scores = tmem + lanes + buffer * kKeys;
                ok = wait(&bars.scores[buffer], (kTiles == 2 ? j : j >> 1) & 1);
                if (!ok) break;
                tc::fence_after();
                const int64_t begin = item.start + int64_t(j) * kKeys;
                // Columns low < c <= high are seen.
                const int high = int(max(int64_t(-1), min(last - begin, int64_t(kKeys))));
                const int low = a.window > 0 ? int(max(int64_t(-1), min(last - a.window - begin, int64_t(kKeys)))) : -1;
                uint32_t hole = 0;
                if (holes[j & 3] == j + 1)
                    for (int i = 0; i < kKeys / kTile; ++i)
                        if (prompt_tile<D>(a, item, int(begin) + i * kTile) < 0) hole |= 1u << i;
                const bool whole = __all_sync(~0u, high >= kKeys - 1 && low < 0 && hole == 0);
                // Scores c .. c + 31, those that are not seen -infinity.
                auto hide = [&](uint32_t (&s)[32], int c) {
                    const int h = min(high - c, 31), l = min(low - c, 31);
                    uint32_t bits = h < 0 ? 0u : (2u << h) - 1u;
                    if (l >= 0) bits &= ~((2u << l) - 1u);
                    if (hole >> (c / kTile) & 1) bits &= 0xFFFF0000u;
                    if (hole >> (c / kTile + 1) & 1) bits &= 0x0000FFFFu;
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i] = bits >> i & 1 ? s[i] : 0xFF800000u;
                };
                uint32_t s[2][32];
                float most = -INFINITY;
                auto maximum = [&](uint32_t (&s)[32], int c) {
                    if (!whole) hide(s, c);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) most = fmaxf(most, fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 1])));
                };
                tc::tmem_load(scores, s[0]);
#pragma unroll 1
                for (int c = 0; c < kKeys; c += 64) {  // 32 columns are on their way while 32 are worked on
                    tc::tmem_wait(s[0]);
                    tc::tmem_load(scores + c + 32, s[1]);
                    maximum(s[0], c);
                    tc::tmem_wait(s[1]);
                    tc::tmem_load(scores + (c + 64) % kKeys, s[0]);
                    maximum(s[1], c + 32);
                }
                most *= to_log2;
                const bool grows = most > top + kPromptLag;
                // One tile's next S may be ready before this block's O is: each phase is waited for in its turn.
                bool waited = j == 0 || kTiles == 2;
                if (__any_sync(~0u, grows)) {
                    const float change = grows ? exp2_approx(top - most) : 1.f;
                    top = grows ? most : top;
                    sum.x *= change;
                    sum.y *= change;
                    if (j > 0) {
                        ok = wait(&bars.sums[tile], (j - 1) & 1);
                        if (!ok) break;
                        waited = true;
                        tc::fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            tc::tmem_load(sums + c, s[1]);
                            tc::tmem_wait(s[1]);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[1][i] = __float_as_uint(__uint_as_float(s[1][i]) * change);
                            tc::tmem_store(sums + c, s[1]);
                        }
                        tc::tmem_load(scores, s[0]);  // again: the wait above was for it too
                    }
                }
                const float against = top == -INFINITY ? 0.f : -top;
                auto weigh = [&](uint32_t (&s)[32], int c) {
                    if (!whole) hide(s, c);
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 z = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(to_log2, to_log2),
                                              make_float2(against, against));
                        const float2 w = make_float2(exp2_approx(z.x), exp2_approx(z.y));
                        sum = add2(sum, w);
                        p[i / 2] = pack2<__half>(w.x, w.y);
                    }
                    tc::tmem_store(scores + c / 2, p);
                };
#pragma unroll 1
                for (int c = 0; c < kKeys; c += 64) {
                    tc::tmem_wait(s[0]);
                    tc::tmem_load(scores + c + 32, s[1]);
                    weigh(s[0], c);
                    tc::tmem_wait(s[1]);
                    if (c + 64 < kKeys) tc::tmem_load(scores + c + 64, s[0]);
                    weigh(s[1], c + 32);
                }
                tc::tmem_stored();
                if (!waited) {
                    ok = wait(&bars.sums[tile], (j - 1) & 1);
                    if (!ok) break;
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(&bars.weights[buffer]);
            }
            if (ok && item.blocks > 0) ok = wait(&bars.sums[tile], (item.blocks - 1) & 1);
            tc::fence_after();
            if (__any_sync(~0u, mine)) {
                uint32_t poison = 0;  // groups whose visible values are not all finite
                if (mine && bad_values) {
                    for (int64_t key = item.start; key <= last; ++key) {
                        if (a.window > 0 && key <= last - a.window) continue;
                        const int64_t at = prompt_tile<D>(a, item, int(key) & ~(kTile - 1));
                        if (at < 0) continue;
#pragma unroll
                        for (int b = 0; b < kGroups; ++b) {
                            const float m = high_bf16(*reinterpret_cast<const uint32_t *>(a.data + at + Tile::pair(true, int(key) & 15, b)));
                            if (m != m) poison |= 1u << b;
                        }
                    }
                }
                const float weight = sum.x + sum.y, per = weight == 0.f ? 0.f : 1.f / (weight * value_factor);
                T *out = static_cast<T *>(a.out) + (int64_t(item.first + token) * a.q_heads + item.head * group + (mine ? index % group : 0)) * D;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t s[32];
                    if (item.blocks > 0) {
                        tc::tmem_load(sums + c, s);
                        tc::tmem_wait(s);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] = 0;
                    }
                    const float by = !ok || (poison >> (c / 64) & 1) ? NAN : per;
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t r[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                r[e] = pack2<T>(__uint_as_float(s[i + 2 * e]) * by, __uint_as_float(s[i + 2 * e + 1]) * by);
                            *reinterpret_cast<uint4 *>(out + c + i) = make_uint4(r[0], r[1], r[2], r[3]);
                        }
                    }
                }
            }
            if (!ok && lane == 0) flag(a.status, SQ_STATUS_TIMEOUT);
        }
    } else if (warp < 12) {
        // Codes into 16-bit operands: a piece of 16 bytes holds four words of one token.
        const int thread = threadIdx.x - 32 * Shape::kSoftmaxWarps;
        constexpr int kPieces = Shape::kPieces, kPerTile = D / 2;  // pieces of a tile's keys or values
        uint4 words[2][kPieces];
        uint32_t pairs[2][kPieces][4];
        // Lane i has the place of tile i of a block, which is looked up a block ahead.
        auto places = [&](int j) {
            const int key = item.start + j * kKeys + lane * kTile;
            const int64_t at = lane < kKeys / kTile && j < item.blocks ? prompt_tile<D>(a, item, key) : 0;
            if (at < 0 && key < item.length) holes[j & 3] = j + 1;
            return at;
        };
        // Key pieces by (token, block of channels, quarter), value pieces by (token, block of 32 bytes, half).
        auto load = [&](int j, int64_t place, bool value) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = (i * Shape::kUnpackThreads + thread) % kPerTile;
                const int part = piece % (D / 32), token = piece / (D / 32);
                const int key = item.start + j * kKeys + (i * Shape::kUnpackThreads + thread) / kPerTile * kTile + token;
                uint4 &w = words[value][i];
                w = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int b = 0; b < 4; ++b) pairs[value][i][b] = 0;
                const int64_t at = __shfl_sync(~0u, place, (i * Shape::kUnpackThreads + thread) / kPerTile);
                if (at < 0) continue;
                const uint8_t *tile = a.data + at;
                const int row = Tile::row(token);
                if (value) {
                    w = *reinterpret_cast<const uint4 *>(tile + Tile::kValues + (part >> 1) * kTile * 32 + token * 32 + (part & 1) * 16);
                } else {
                    constexpr int kParts = Tile::kBlockRow / 16;  // pieces of a block's row
                    w = *reinterpret_cast<const uint4 *>(tile + (part / kParts) * kTile * Tile::kBlockRow + row * Tile::kBlockRow + (part % kParts) * 16);
                }
                if (key < item.length) {
                    const uint32_t *from = reinterpret_cast<const uint32_t *>(tile + (value ? Tile::kValuePairs : Tile::kKeyPairs)) + row * kGroups;
                    if (D == 64) {
                        pairs[value][i][0] = from[0];
                    } else if (D == 128 || !value) {
                        const uint2 p = *reinterpret_cast<const uint2 *>(from + (value ? 0 : part / 4 * 2));
                        pairs[value][i][0] = p.x, pairs[value][i][1] = p.y;
                    } else {
                        const uint4 p = *reinterpret_cast<const uint4 *>(from);
                        pairs[value][i][0] = p.x, pairs[value][i][1] = p.y, pairs[value][i][2] = p.z, pairs[value][i][3] = p.w;
                    }
                }
            }
        };
        auto write = [&](uint8_t *to, uint8_t *more, bool value) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = (i * Shape::kUnpackThreads + thread) % kPerTile;
                const int part = piece % (D / 32), token = piece / (D / 32);
                const int row = (i * Shape::kUnpackThreads + thread) / kPerTile * kTile + token;  // key of the block
                const uint32_t w[4] = {words[value][i].x, words[value][i].y, words[value][i].z, words[value][i].w};
                if (!value && part % 4 == 0) {  // groups part / 4 * 2 and, if there is one, the next: m, m, 8 s, 8 s
                    uint32_t r[4] = {};
#pragma unroll
                    for (int b = 0; b < (kGroups < 2 ? 1 : 2); ++b) {
                        const float s = low_bf16(pairs[value][i][b]) * (8 / kKeyDivisor), m = high_bf16(pairs[value][i][b]) / kKeyDivisor;
                        r[2 * b] = pack2<__half>(m, m);
                        r[2 * b + 1] = pack2<__half>(s, s);
                    }
                    uint8_t *const from = more + row * 16;
                    *reinterpret_cast<uint4 *>(from + part / 4 * kKeys * 16) = make_uint4(r[0], r[1], r[2], r[3]);
                    if (D < 256) *reinterpret_cast<uint4 *>(from + kKeys * 16) = make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // Channels 8 oct + 0..7 of group g; its pair is the piece's pair number p.
                    int g, oct, p;
                    if (value) {
                        const int number = part * 4 + e;
                        g = number % kGroups, oct = number / kGroups;
                        p = e % kGroups;
                    } else if (D == 64) {
                        g = 0, oct = 4 * part + e, p = 0;
                    } else {
                        p = e >> 1, g = part / 4 * 2 + p, oct = 2 * (part & 3) + (e & 1);
                    }
                    uint32_t pair = pairs[value][i][p];
                    uint4 x;
                    if (value) {
                        if (high_bf16(pair) != high_bf16(pair)) pair = 0, bad_values = 1;
                        x = unpack_f16(w[e], __float2half2_rn(low_bf16(pair) * value_factor), __float2half2_rn(high_bf16(pair) * value_factor));
                    } else {
                        x = unpack_middle(w[e], __float2half2_rn(low_bf16(pair) / kKeyDivisor));
                    }
                    *reinterpret_cast<uint4 *>(to + g * kKeys * 128 + row * 128 + ((oct ^ (row & 7)) << 4)) = x;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
        };
        int64_t place = places(0), next_place;
        if (item.blocks > 0) load(0, place, false);
#pragma unroll 1
        for (int j = 0; j < item.blocks; ++j) {
            const int stage = j & 1;
            load(j, place, true);
            next_place = places(j + 1);
            if (j > 1 && !wait(&bars.keys_free[stage], ((j >> 1) - 1) & 1)) break;
            write(keys + stage * Shape::kKeyBytes, more_keys + stage * Shape::kMoreKey, false);
            if (lane == 0) tc::bar_arrive(&bars.keys[stage]);
            place = next_place;
            if (j + 1 < item.blocks) load(j + 1, place, false);
            if (j > 1 && !wait(&bars.values_free[stage], ((j >> 1) - 1) & 1)) break;
            write(values + stage * Shape::kKeyBytes, nullptr, true);
            if (lane == 0) tc::bar_arrive(&bars.values[stage]);
        }
    } else if (lane == 0) {
        constexpr uint32_t kScores = tc::half_product(kKeys, false, false), kSums = tc::half_product(D, false, true);
        auto scores = [&](int tile, int buffer, int stage) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                tc::mma_half(tmem + buffer * kKeys, tc::operand(tc::smem_u32(queries + tile * Shape::kQueryBytes + (k >> 2) * 16384) + (k & 3) * 32),
                             tc::operand(tc::smem_u32(keys + stage * Shape::kKeyBytes + (k >> 2) * kKeys * 128) + (k & 3) * 32), kScores, k > 0);
            tc::mma_half(tmem + buffer * kKeys, tc::operand_narrow(tc::smem_u32(more_queries + tile * Shape::kMoreQuery), 128 * 16),
                         tc::operand_narrow(tc::smem_u32(more_keys + stage * Shape::kMoreKey), kKeys * 16), kScores, true);
            tc::mma_commit(&bars.scores[buffer]);
        };
        bool ok = item.blocks == 0 || wait_alone(&bars.query, 0);
        // The keys of block j, and its products with the queries of each tile.
        auto begin = [&](int j, int tile) {
            const int stage = j & 1;
            if (tile == 0) ok = ok && wait_alone(&bars.keys[stage], (j >> 1) & 1);
            if (!ok) return;
            tc::fence_after();
            scores(tile, kTiles == 2 ? tile : stage, stage);
            if (tile == live - 1) tc::mma_commit(&bars.keys_free[stage]);
        };
        for (int tile = 0; tile < live && item.blocks > 0; ++tile) begin(0, tile);
        for (int j = 0; j < item.blocks && ok; ++j) {
            const int stage = j & 1;
            if (kTiles == 1 && j + 1 < item.blocks) begin(j + 1, 0);
            for (int tile = 0; tile < live && ok; ++tile) {
                const int buffer = kTiles == 2 ? tile : stage;
                if (tile == 0) ok = wait_alone(&bars.values[stage], (j >> 1) & 1);
                ok = ok && wait_alone(&bars.weights[buffer], (kTiles == 2 ? j : j >> 1) & 1);
                if (!ok) break;
                tc::fence_after();
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    tc::mma_half_tmem(tmem + Shape::kColumnsO + tile * D, tmem + buffer * kKeys + k * 8,
                                      tc::operand_mn(tc::smem_u32(values + stage * Shape::kKeyBytes + k * 2048), kKeys * 128), kSums, j > 0 || k > 0);
                tc::mma_commit(&bars.sums[tile]);
                if (tile == live - 1) tc::mma_commit(&bars.values_free[stage]);
                if (kTiles == 2 && j + 1 < item.blocks) begin(j + 1, tile);
            }
        }
        if (!ok) {  // the products that were issued end before the tensor memory is freed
            int alone = 0;
            tc::mma_commit(&bars.end);
            tc::bar_wait(&bars.end, 0, &alone, tc::kWaitClocks);
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 12) tc::tmem_free(tmem, 512);
}

template <class T, int D>
cudaError_t launch_prompt(const sq_kv_attention_args &a, int few_rows, cudaStream_t s) {
    using Shape = PromptShape<D>;
    const int per = Shape::kTiles * 128 / (a.q_heads / a.heads);
    const unsigned strips = unsigned(a.tokens / per + a.num_seqs);
    const int64_t grid = int64_t(strips) * a.heads;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const cudaError_t e = cudaFuncSetAttribute(prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kShared);
    if (e != cudaSuccess) return e;
    prompt_kernel<T, D><<<unsigned(grid), kPromptThreads, Shape::kShared, s>>>(a, per, strips, few_rows);
    return cudaGetLastError();
}

}  // namespace

// Sequences with more than `few_rows` rows (new tokens times query heads of a kv head, at most 128 of
// these); cu_seqlens given.
cudaError_t launch_prompt_attention(const sq_kv_attention_args &a, int few_rows, cudaStream_t s) {
    if (a.dtype == SQ_BF16) {
        switch (a.dim) {
            case 64: return launch_prompt<__nv_bfloat16, 64>(a, few_rows, s);
            case 128: return launch_prompt<__nv_bfloat16, 128>(a, few_rows, s);
            default: return launch_prompt<__nv_bfloat16, 256>(a, few_rows, s);
        }
    }
    switch (a.dim) {
        case 64: return launch_prompt<__half, 64>(a, few_rows, s);
        case 128: return launch_prompt<__half, 128>(a, few_rows, s);
        default: return launch_prompt<__half, 256>(a, few_rows, s);
    }
}

}  // namespace sq
