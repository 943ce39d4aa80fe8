// Attention of prompts over the paged 4-bit cache, on tcgen05 (sq_attention.cu has few rows).
//
// A CTA takes 256 query rows of one kv head, (token, query head) pairs, in two tiles of
// 128 (heads of 256 channels: one tile, as its sums fill the tensor memory), and walks
// the keys in blocks of 128 (64).  Per block:
//   eight warps (four for heads of 64) write out the codes as 16-bit keys and values in
//   shared memory, two to four blocks ahead,
//   one warp issues S = Q K^T and O += P V, S, P and O in tensor memory,
//   four warps a tile, a thread to a row, turn S into P, which overwrites it.
// While a tile's S becomes P, the other tile's products run (one tile: S and P have two
// buffers).  Products of 128 x 64 take as long as those of 128 x 128, 64 clocks.
// Scores take keys as they are held: s (c - 8) has 3 + 8 significant bits and so is an f16,
// and the rest of a group, m + 8 s, meets the sum of the query's channels in one more step
// of K (the sum's f16 and its remainder, each by m and by 8 s).  Queries are f16 with each
// row's largest value near 2^8.  Values m + s c and weights are rounded to f16 too, whatever
// the cache's type (bf16 values and weights were half as exact: 2.6e-3 of an output's norm,
// of which 1.7e-3 are its own rounding).  Keys and values are times a power of two each that
// brings the largest of the item's to 2^13 .. 2^15, which a scan of scales and minima finds
// first: f16 then keeps a key exactly down to 2^-24 of the largest.
// Row maxima may lag by 2^8, so sums in tensor memory are seldom rescaled.
//
// 4096 tokens over 16384 of 32 / 8 heads of 128: 1103 us, 870 TFLOP/s, 0.52 of the burst
// rate of a library product.  A tile's chain bounds it (products, a commit, S read, maxima,
// weights stored, an arrival), of which the other tile's products hide half; blocks of 64
// keys with S and P in two buffers measured 1371 us, as a product of 128 x 64 takes the 64
// clocks of one of 128 x 128.
#include "sq_kv.cuh"
#include "sq_rows.cuh"
#include "sq_tc.cuh"
#include "sq_vec.cuh"

namespace sq {
namespace {

constexpr int kKeyPower = 13, kValuePower = 14;  // of the largest |m| + 15 s of an item's keys and values
constexpr float kPromptLag = 8.f;
// Weights are 2^kPromptLift over what the maximum would make them, 2^15 at most: f16 then drops those below 2^-32 of
// the row's largest and not those below 2^-25, which count where the largest belong to keys without a value.
constexpr float kPromptLift = 7.f;

template <int D>
struct PromptShape {
    using Tile = KvTile<D>;
    static constexpr int kTiles = D == 256 ? 1 : 2;             // of 128 rows
    static constexpr int kKeys = D == 256 ? 64 : 128;           // of a block
    static constexpr int kBuffers = D == 256 ? 2 : 1;           // of S and P for a tile
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr int kSoftmaxWarps = 4 * kTiles, kUnpackWarps = D == 64 ? 4 : 8, kProductWarp = kSoftmaxWarps + kUnpackWarps;
    static constexpr int kUnpackThreads = 32 * kUnpackWarps, kThreads = 32 * (kProductWarp + 4);
    // With 128 keys a softmax thread holds 128 scores: the registers that 16 or 20 warps are launched with
    // are shared out anew, and what the three roles take is no more than that.
    static constexpr bool kShare = kKeys == 128;
    static constexpr int kLaunchRegisters = D == 128 ? 96 : 128;
    static constexpr int kSoftmaxRegisters = D == 128 ? 160 : 168, kUnpackRegisters = D == 128 ? 56 : 96, kProductRegisters = D == 128 ? 48 : 48;
    static_assert(!kShare || 32 * (kSoftmaxWarps * kSoftmaxRegisters + kUnpackWarps * kUnpackRegisters + 4 * kProductRegisters) <=
                                 kThreads * kLaunchRegisters, "");
    static constexpr int kQueryBytes = 128 * D * 2, kKeyBytes = kKeys * D * 2;
    static constexpr int kMoreQuery = 128 * 32, kMoreKey = kKeys * 32;  // the last step of K: 16 values a row
    static constexpr int kShared = kTiles * (kQueryBytes + kMoreQuery) + kStages * (2 * kKeyBytes + kMoreKey) + 1024;
    static constexpr int kColumnsO = kTiles * kBuffers * kKeys; // S, P: [0, kColumnsO)
    static constexpr int kPieces = kKeys * D / 32 / kUnpackThreads;  // 16-byte pieces of a block's keys for a thread
    static_assert(kColumnsO + kTiles * D <= 512 && kPieces * kUnpackThreads * 32 == kKeys * D && kShared <= 227 * 1024, "");
    static_assert((kStages & (kStages - 1)) == 0 && kStages <= 4, "");
};

struct PromptBars {
    uint64_t query, keys[4], keys_free[4], values[4], values_free[4];  // by stage
    uint64_t scores[2], weights[2];                                    // by tile, or by block modulo 2
    uint64_t sums[4];                                                  // by tile and block modulo 2
    uint64_t end;
};

// Codes of 8 channels as f16 pairs (c - 8) s, exactly: in the top of the mantissa a code makes 16 + c, and
// 24 s has 10 significant bits.
__device__ __forceinline__ uint4 unpack_middle(uint32_t w, __half2 s, __half2 less_24s) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = and_or(i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6), 0x03C003C0u, 0x4C004C00u);
        const __half2 v = __hfma2(reinterpret_cast<const __half2 &>(x), s, less_24s);
        r[i] = reinterpret_cast<const uint32_t &>(v);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
// Codes of 8 channels as f16 pairs c s + m: 1024 + c and, from the next four bits, 1024 + 16 c, less 1024.
__device__ __forceinline__ uint4 unpack_value(uint32_t w, __half2 s, __half2 s16, __half2 m) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = and_or(i < 2 ? w : w >> 8, i & 1 ? 0x00F000F0u : 0x000F000Fu, 0x64006400u), base = 0x64006400u;
        const __half2 c = __hsub2(reinterpret_cast<const __half2 &>(x), reinterpret_cast<const __half2 &>(base));
        const __half2 v = __hfma2(c, i & 1 ? s16 : s, m);
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
__global__ void __launch_bounds__(PromptShape<D>::kThreads, 1) prompt_kernel(sq_kv_attention_args a, int tokens_per_item, unsigned strips, int few_rows) {
    using Shape = PromptShape<D>;
    using Tile = KvTile<D>;
    constexpr int kTiles = Shape::kTiles, kKeys = Shape::kKeys, kBuffers = Shape::kBuffers, kStages = Shape::kStages, kGroups = Tile::kGroups;
    extern __shared__ uint8_t raw[];
    __shared__ PromptBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, bad_values;
    __shared__ unsigned most_key, most_value;
    __shared__ volatile int holes[8];  // block + 1 of the last one with tiles to leave out, by block modulo 8
    uint8_t *const queries = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t *const keys = queries + kTiles * Shape::kQueryBytes, *const values = keys + kStages * Shape::kKeyBytes;
    uint8_t *const more_queries = values + kStages * Shape::kKeyBytes, *const more_keys = more_queries + kTiles * Shape::kMoreQuery;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.q_heads / a.heads;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the few rows' kernel, once every CTA has begun

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
        const int tokens = int(min(item.count - token, int64_t(tokens_per_item)));
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

    if (warp == Shape::kProductWarp) {
        tc::tmem_alloc(&tmem_slot, 512);
        if (lane == 0) {
            tc::bar_init(&bars.query, 4 * live);
            for (int i = 0; i < 4; ++i) {
                tc::bar_init(&bars.keys[i], Shape::kUnpackWarps);
                tc::bar_init(&bars.values[i], Shape::kUnpackWarps);
                tc::bar_init(&bars.keys_free[i], 1);
                tc::bar_init(&bars.values_free[i], 1);
                tc::bar_init(&bars.sums[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                tc::bar_init(&bars.scores[i], 1);
                tc::bar_init(&bars.weights[i], 4);
            }
            tc::bar_init(&bars.end, 1);
            tc::bar_init_fence();
            abort_flag = 0;
            bad_values = 0;
            most_key = most_value = 0;
            for (int i = 0; i < 8; ++i) holes[i] = 0;
        }
        __syncwarp();
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_slot;

    // Largest |m| + 15 s of the item's keys and values.
    {
        constexpr int kEach = D / 16;  // accesses of four pairs a tile, of keys and of values
        const int64_t end = min(int64_t(item.start) + int64_t(item.blocks) * kKeys, int64_t(item.length));
        float key_most = 0.f, value_most = 0.f;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < (end - item.start + kTile - 1) / kTile * kEach; i += Shape::kThreads) {
            const int key = item.start + int(i / kEach) * kTile, first = int(i % kEach) * 4;
            const int64_t at = prompt_tile<D>(a, item, key);
            if (at < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4 *>(a.data + at + Tile::kKeyPairs + first * 4);
            const uint4 y = *reinterpret_cast<const uint4 *>(a.data + at + Tile::kValuePairs + first * 4);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = (first + e) / kGroups, token = (row & 8) | ((row & 1) << 2) | ((row >> 1) & 3);
                if (key + token < item.length) {
                    key_most = fmaxf(key_most, fabsf(high_bf16(w[e])) + 15.f * low_bf16(w[e]));
                    value_most = fmaxf(value_most, fabsf(high_bf16(v[e])) + 15.f * low_bf16(v[e]));
                }
            }
        }
        const unsigned k = __reduce_max_sync(~0u, __float_as_uint(fminf(key_most, 3e38f)));
        const unsigned v = __reduce_max_sync(~0u, __float_as_uint(fminf(value_most, 3e38f)));
        if (lane == 0) {
            atomicMax(&most_key, k);
            atomicMax(&most_value, v);
        }
        __syncthreads();
    }
    const int value_shift = most_value == 0 ? 0 : min(126, kValuePower - (int(most_value >> 23) - 127));  // -114 at least
    const float value_factor = __uint_as_float(uint32_t(127 + value_shift) << 23);
    const int key_shift = most_key == 0 ? 0 : min(126, kKeyPower - (int(most_key >> 23) - 127));  // -115 at least
    const float key_factor = __uint_as_float(uint32_t(127 + key_shift) << 23);
    // Of a whole warp: all lanes go on, or none does.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        return bool(__all_sync(~0u, tc::bar_wait_or_look(bar, parity, &abort_flag, a.wait_clocks)));
    };

    float top = -INFINITY;  // of a row
    float2 sum = make_float2(0.f, 0.f);  // of its weights, in two parts
    if (warp < Shape::kSoftmaxWarps) {
        if constexpr (Shape::kShare) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(Shape::kSoftmaxRegisters));
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
            // At least what scores of up to 2^33 vanish under: zero would make a hidden one's -infinity a NaN.
            const float to_log2 = fmaxf(ldexpf(a.scale * kLog2e, -shift - key_shift), 0x1p-100f);
            const int64_t last = mine ? min(item.before + token, int64_t(item.length) - 1) : -1;
            // Columns low < c <= high of the keys from item.start on are seen; the warp sees blocks whole_from to
            // whole_to - 1 whole.
            const int high = int(max(int64_t(-1), last - item.start));
            // (The window is of the token's own position, which may lie past the table.)
            const int low = a.window > 0 ? int(max(int64_t(-1), min(item.before + token - a.window - item.start, int64_t(item.length)))) : -1;
            const int whole_from = __reduce_max_sync(~0u, (low + kKeys) / kKeys), whole_to = __reduce_min_sync(~0u, (high + 1) / kKeys);
            const uint32_t lanes = uint32_t(warp & 3) << 21;
            const uint32_t sums = tmem + lanes + Shape::kColumnsO + tile * D;
            bool ok = true;
            for (int j = 0; j < item.blocks && ok; ++j) {
                const int buffer = kBuffers == 2 ? j & 1 : tile;
                const uint32_t scores = tmem + lanes + buffer * kKeys;
                ok = wait(&bars.scores[buffer], (kBuffers == 2 ? j >> 1 : j) & 1);
                if (!ok) break;
                tc::fence_after();
                uint32_t s[kKeys / 32][32];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) tc::tmem_load(scores + 32 * c, s[c]);
                const bool holed = holes[j & 7] == j + 1, whole = j >= whole_from && j < whole_to && !holed;
                uint32_t hole = 0;
                if (holed)
                    for (int i = 0; i < kKeys / kTile; ++i)
                        if (prompt_tile<D>(a, item, item.start + j * kKeys + i * kTile) < 0) hole |= 1u << i;
                // Scores c .. c + 31, those that are not seen -infinity.
                auto hide = [&](uint32_t (&s)[32], int c) {
                    const int h = min(high - j * kKeys - c, 31), l = min(low - j * kKeys - c, 31);
                    uint32_t bits = h < 0 ? 0u : (2u << h) - 1u;
                    if (l >= 0) bits &= ~((2u << l) - 1u);
                    if (hole >> (c / kTile) & 1) bits &= 0xFFFF0000u;
                    if (hole >> (c / kTile + 1) & 1) bits &= 0x0000FFFFu;
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i] = bits >> i & 1 ? s[i] : 0xFF800000u;
                };
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) tc::tmem_wait(s[c]);
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) hide(s[c], 32 * c);
                }
                float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        part[c % 4] = max3(part[c % 4], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                const float most = fmaxf(max3(part[0], part[1], part[2]), part[3]) * to_log2;
                const bool grows = most > top + kPromptLag;
                if (__any_sync(~0u, grows)) {
                    const float change = grows ? exp2_approx(top - most) : 1.f;
                    top = grows ? most : top;
                    sum.x *= change;
                    sum.y *= change;
                    if (j > 0) {
                        // This block's S was ready after the O of two blocks before: that barrier's last phase is over.
                        ok = wait(&bars.sums[2 * tile + ((j - 1) & 1)], ((j - 1) >> 1) & 1);
                        if (!ok) break;
                        tc::fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tc::tmem_load(sums + c, o);
                            tc::tmem_wait(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * change);
                            tc::tmem_store(sums + c, o);
                        }
                    }
                }
                const float against = top == -INFINITY ? 0.f : kPromptLift - top;
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 z = fma2(make_float2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), make_float2(to_log2, to_log2),
                                              make_float2(against, against));
                        const float2 w = make_float2(exp2_approx(z.x), exp2_approx(z.y));
                        sum = add2(sum, w);
                        p[i / 2] = pack2<__half>(w.x, w.y);
                    }
                    tc::tmem_store(scores + c * 16, p);
                }
                tc::tmem_stored();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(&bars.weights[buffer]);
            }
            if (ok && item.blocks > 0) ok = wait(&bars.sums[2 * tile + ((item.blocks - 1) & 1)], ((item.blocks - 1) >> 1) & 1);
            tc::fence_after();
            if (__any_sync(~0u, mine)) {
                uint32_t poison = 0;  // groups whose visible values are not all finite
                if (mine && bad_values) {
                    for (int64_t key = item.start; key <= last; ++key) {
                        if (a.window > 0 && key <= item.before + token - a.window) continue;
                        const int64_t at = prompt_tile<D>(a, item, int(key) & ~(kTile - 1));
                        if (at < 0) continue;
#pragma unroll
                        for (int b = 0; b < kGroups; ++b) {
                            const float m = high_bf16(*reinterpret_cast<const uint32_t *>(a.data + at + Tile::pair(true, int(key) & 15, b)));
                            if (m != m) poison |= 1u << b;
                        }
                    }
                }
                // The values' factor apart: its product with the weights' sum may leave fp32.
                const float weight = sum.x + sum.y, per = weight == 0.f ? 0.f : 1.f / weight;
                const float back = __uint_as_float(uint32_t(127 - value_shift) << 23);
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
                                r[e] = pack2<T>(__uint_as_float(s[i + 2 * e]) * by * back, __uint_as_float(s[i + 2 * e + 1]) * by * back);
                            *reinterpret_cast<uint4 *>(out + c + i) = make_uint4(r[0], r[1], r[2], r[3]);
                        }
                    }
                }
            }
            if (!ok && lane == 0) flag(a.status, SQ_STATUS_TIMEOUT);
        }
    } else if (warp < Shape::kProductWarp) {
        if constexpr (Shape::kShare) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Shape::kUnpackRegisters));
        // Codes into 16-bit operands: a piece of 16 bytes holds four words of one token.
        // Piece i of this thread: tile tile0 + i kSpan of a block, the same token and part of it for all i.
        // Key pieces go by (token, block of channels, quarter), value pieces by (token, block of 32 bytes, half).
        constexpr int kPieces = Shape::kPieces, kPerTile = D / 2, kSpan = Shape::kUnpackThreads / kPerTile;
        const int thread = threadIdx.x - 32 * Shape::kSoftmaxWarps;
        const int tile0 = thread / kPerTile, part = thread % (D / 32), token = thread % kPerTile / (D / 32), row = Tile::row(token);
        constexpr int kParts = Tile::kBlockRow / 16, kKeyGroups = Tile::kBlockGroups;  // pieces of a block's row; groups of a key piece
        constexpr int kValueGroups = kGroups;
        const int key_at = (part / kParts) * kTile * Tile::kBlockRow + row * Tile::kBlockRow + (part % kParts) * 16;
        const int key_pair_at = Tile::kKeyPairs + (row * kGroups + (D == 256 ? part / 4 * 2 : 0)) * 4;
        const int value_at = Tile::kValues + (part >> 1) * kTile * 32 + token * 32 + (part & 1) * 16;
        const int value_pair_at = Tile::kValuePairs + row * kGroups * 4;
        // Where a piece's word e, 8 channels, goes in an operand of rows of 64 channels: the first one's place,
        // other 16 bytes of the row (the swizzle is an exclusive or) or another group.
        const uint32_t row0 = uint32_t(tile0 * kTile + token), swizzle = token & 7;
        const uint32_t key_to = tc::smem_u32(keys) + (D == 256 ? part / 4 * 2 : 0) * kKeys * 128 + row0 * 128 +
                                (((D == 64 ? 4 * part : 2 * (part & 3)) ^ swizzle) << 4);
        const uint32_t value_to = tc::smem_u32(values) + row0 * 128 + (((D == 256 ? part : D == 128 ? 2 * part : 4 * part) ^ swizzle) << 4);
        auto key_word = [&](uint32_t at, int e) { return D == 64 ? at ^ (e << 4) : (at ^ ((e & 1) << 4)) + (e >> 1) * kKeys * 128; };
        auto value_word = [&](uint32_t at, int e) {
            return D == 64 ? at ^ (e << 4) : D == 128 ? (at ^ ((e >> 1) << 4)) + (e & 1) * kKeys * 128 : at + e * kKeys * 128;
        };
        const uint32_t more_to = tc::smem_u32(more_keys) + row0 * 16 + part / 4 * kKeys * 16;
        auto put = [](uint32_t to, uint4 x) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
        };
        uint4 key_words[kPieces], value_words[kPieces];
        uint32_t key_pairs[kPieces][kKeyGroups], value_pairs[kPieces][kValueGroups];
        // Lane i has the place of tile i of a block, which is looked up a block ahead.
        auto places = [&](int j) {
            const int key = item.start + j * kKeys + lane * kTile;
            const int64_t at = lane < kKeys / kTile && j < item.blocks ? prompt_tile<D>(a, item, key) : 0;
            if (at < 0 && key < item.length) holes[j & 7] = j + 1;
            return at;
        };
        auto load_keys = [&](int j, int64_t place) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int64_t at = __shfl_sync(~0u, place, tile0 + i * kSpan);
                const uint8_t *tile = a.data + at;
                key_words[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int b = 0; b < kKeyGroups; ++b) key_pairs[i][b] = 0;
                if (at >= 0) {
                    key_words[i] = *reinterpret_cast<const uint4 *>(tile + key_at);
                    if (item.start + j * kKeys + (tile0 + i * kSpan) * kTile + token < item.length) {
                        if (D == 64) {
                            key_pairs[i][0] = *reinterpret_cast<const uint32_t *>(tile + key_pair_at);
                        } else {
                            const uint2 p = *reinterpret_cast<const uint2 *>(tile + key_pair_at);
                            key_pairs[i][0] = p.x, key_pairs[i][kKeyGroups - 1] = p.y;
                        }
                    }
                }
            }
        };
        auto load_values = [&](int j, int64_t place) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int64_t at = __shfl_sync(~0u, place, tile0 + i * kSpan);
                const uint8_t *tile = a.data + at;
                value_words[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int b = 0; b < kValueGroups; ++b) value_pairs[i][b] = 0;
                if (at >= 0) {
                    value_words[i] = *reinterpret_cast<const uint4 *>(tile + value_at);
                    if (item.start + j * kKeys + (tile0 + i * kSpan) * kTile + token < item.length) {
#pragma unroll
                        for (int b = 0; b < kValueGroups; ++b)
                            value_pairs[i][b] = reinterpret_cast<const uint32_t *>(tile + value_pair_at)[b];
                    }
                }
            }
        };
        auto write_keys = [&](int stage) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t at = key_to + stage * Shape::kKeyBytes + i * kSpan * kTile * 128;
                const uint32_t w[4] = {key_words[i].x, key_words[i].y, key_words[i].z, key_words[i].w};
                __half2 s[kKeyGroups], less[kKeyGroups];
#pragma unroll
                for (int b = 0; b < kKeyGroups; ++b) {
                    const float scale = low_bf16(key_pairs[i][b]) * key_factor;
                    s[b] = __float2half2_rn(scale);
                    less[b] = __float2half2_rn(-24.f * scale);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int b = D == 64 ? 0 : e >> 1;
                    put(key_word(at, e), unpack_middle(w[e], s[b % kKeyGroups], less[b % kKeyGroups]));
                }
                if (part % 4 == 0) {  // groups part / 4 * 2 and, if there is one, the next: m, m, 8 s, 8 s
                    const uint32_t more = more_to + stage * Shape::kMoreKey + i * kSpan * kTile * 16;
                    uint32_t r[4] = {};
#pragma unroll
                    for (int b = 0; b < kKeyGroups; ++b) {
                        const float m = high_bf16(key_pairs[i][b]) * key_factor, s8 = low_bf16(key_pairs[i][b]) * key_factor * 8.f;
                        r[2 * b] = pack2<__half>(m, m);
                        r[2 * b + 1] = pack2<__half>(s8, s8);
                    }
                    put(more, make_uint4(r[0], r[1], r[2], r[3]));
                    if (D < 256) put(more + kKeys * 16, make_uint4(0, 0, 0, 0));
                }
            }
        };
        auto write_values = [&](int stage) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t at = value_to + stage * Shape::kKeyBytes + i * kSpan * kTile * 128;
                const uint32_t w[4] = {value_words[i].x, value_words[i].y, value_words[i].z, value_words[i].w};
                __half2 s[kValueGroups], s16[kValueGroups], m[kValueGroups];
#pragma unroll
                for (int b = 0; b < kValueGroups; ++b) {
                    uint32_t pair = value_pairs[i][b];
                    if ((pair & 0x7FFFFFFFu) > 0x7F800000u) pair = 0, bad_values = 1;  // m is NaN
                    s[b] = __float2half2_rn(low_bf16(pair) * value_factor);
                    s16[b] = __float2half2_rn(low_bf16(pair) * (value_factor / 16));
                    m[b] = __float2half2_rn(high_bf16(pair) * value_factor);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) put(value_word(at, e), unpack_value(w[e], s[e % kValueGroups], s16[e % kValueGroups], m[e % kValueGroups]));
            }
        };
        auto written = [&](uint64_t *bar) {
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::bar_arrive(bar);
        };
        int64_t place = places(0), next_place;
        if (item.blocks > 0) load_keys(0, place);
#pragma unroll 1
        for (int j = 0; j < item.blocks; ++j) {
            const int stage = j % kStages;
            load_values(j, place);
            next_place = places(j + 1);
            if (j >= kStages && !wait(&bars.keys_free[stage], (j / kStages - 1) & 1)) break;
            write_keys(stage);
            written(&bars.keys[stage]);
            place = next_place;
            if (j + 1 < item.blocks) load_keys(j + 1, place);
            if (j >= kStages && !wait(&bars.values_free[stage], (j / kStages - 1) & 1)) break;
            write_values(stage);
            written(&bars.values[stage]);
        }
    } else {
        if constexpr (Shape::kShare) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Shape::kProductRegisters));
        if (warp == Shape::kProductWarp) {
        constexpr uint32_t kScores = tc::half_product(kKeys, false), kSums = tc::half_product(D, true);
        // Descriptors of the first operands; others are further by bytes / 16.
        const uint64_t query = tc::operand(tc::smem_u32(queries)), key = tc::operand(tc::smem_u32(keys));
        const uint64_t value = tc::operand_mn(tc::smem_u32(values), kKeys * 128);
        const uint64_t more_query = tc::operand_narrow(tc::smem_u32(more_queries), 128 * 16);
        const uint64_t more_key = tc::operand_narrow(tc::smem_u32(more_keys), kKeys * 16);
        // The same for all lanes, and known to be: operands stay in uniform registers.
        const uint32_t base = __shfl_sync(~0u, tmem, 0);
        const int blocks = __shfl_sync(~0u, item.blocks, 0), tiles = __shfl_sync(~0u, live, 0);
        bool ok = blocks == 0 || wait(&bars.query, 0);
        // Not formed ahead of the loop, each operand of a block in registers of its own.
        auto here = [](uint64_t x) {
            asm volatile("" : "+l"(x));
            return x;
        };
        // S of block j for a tile.
        auto begin = [&](int j, int tile) {
            const int stage = j % kStages, buffer = kBuffers == 2 ? j & 1 : tile;
            if (tile == 0) ok = ok && wait(&bars.keys[stage], (j / kStages) & 1);
            if (!ok) return;
            tc::fence_after();
            const uint64_t q = here(query) + tile * (Shape::kQueryBytes / 16), k = here(key) + stage * (Shape::kKeyBytes / 16);
            const uint64_t more = here(more_key) + stage * (Shape::kMoreKey / 16);
            if (tc::elected()) {
                const uint32_t d = base + buffer * kKeys;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    tc::mma_half(d, q + ((i >> 2) * 16384 + (i & 3) * 32) / 16, k + ((i >> 2) * kKeys * 128 + (i & 3) * 32) / 16, kScores, i > 0);
                tc::mma_half(d, here(more_query) + tile * (Shape::kMoreQuery / 16), more, kScores, true);
                tc::mma_commit(&bars.scores[buffer]);
                if (tile == tiles - 1) tc::mma_commit(&bars.keys_free[stage]);
            }
            __syncwarp();
        };
        for (int tile = 0; tile < tiles && blocks > 0; ++tile) begin(0, tile);
#pragma unroll 1
        for (int j = 0; j < blocks && ok; ++j) {
            const int stage = j % kStages;
            if (kBuffers == 2 && j + 1 < blocks) begin(j + 1, 0);
            ok = ok && wait(&bars.values[stage], (j / kStages) & 1);
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                if (tile >= tiles || !ok) break;
                const int buffer = kBuffers == 2 ? j & 1 : tile;
                ok = wait(&bars.weights[buffer], (kBuffers == 2 ? j >> 1 : j) & 1);
                if (!ok) break;
                tc::fence_after();
                const uint64_t v = here(value) + stage * (Shape::kKeyBytes / 16);
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        tc::mma_half_tmem(base + Shape::kColumnsO + tile * D, base + buffer * kKeys + k * 8, v + k * 2048 / 16, kSums, j > 0 || k > 0);
                    tc::mma_commit(&bars.sums[2 * tile + (j & 1)]);
                    if (tile == tiles - 1) tc::mma_commit(&bars.values_free[stage]);
                }
                __syncwarp();
                if (kBuffers == 1 && j + 1 < blocks) begin(j + 1, tile);
            }
        }
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == Shape::kProductWarp) {
        if (*static_cast<volatile int *>(&abort_flag)) {  // a role gave up: the products that were issued end first
            int alone = 0;
            if (tc::elected()) tc::mma_commit(&bars.end);
            __syncwarp();
            tc::bar_wait(&bars.end, 0, &alone, tc::kWaitClocks);
        }
        tc::tmem_free(tmem, 512);
    }
}

template <class T, int D>
cudaError_t launch_prompt(const sq_kv_attention_args &a, int few_rows, cudaStream_t s) {
    using Shape = PromptShape<D>;
    const int per = Shape::kTiles * 128 / (a.q_heads / a.heads);
    const unsigned strips = unsigned(a.tokens / per + a.num_seqs);
    const int64_t grid = int64_t(strips) * a.heads;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = allow_shared(prompt_kernel<T, D>, Shape::kShared, devices);
    if (e != cudaSuccess) return e;
    if (Shape::kShare) {
        // A warp that asks for more registers than the block was launched with and others gave back waits for ever:
        // what the compiler allotted (in eights) is what the shares were added up against, or nothing is launched.
        static std::atomic<int> registers{0};
        if (registers.load(std::memory_order_relaxed) == 0) {
            cudaFuncAttributes attributes;
            e = cudaFuncGetAttributes(&attributes, prompt_kernel<T, D>);
            if (e != cudaSuccess) return e;
            registers.store((attributes.numRegs + 7) / 8 * 8, std::memory_order_relaxed);
        }
        if (registers.load(std::memory_order_relaxed) < Shape::kLaunchRegisters) return cudaErrorInvalidKernelImage;
    }
    prompt_kernel<T, D><<<unsigned(grid), Shape::kThreads, Shape::kShared, s>>>(a, per, strips, few_rows);
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
