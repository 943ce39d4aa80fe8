// Angles of rotary positions, and the form of the 4-bit cache, shared by the
// rotation, the cache's append and read, and the attention over it.
#pragma once

#include "sq_common.cuh"

namespace sq {

// The angle position * frequency as a fraction of a turn in units of 2^-64: a product of
// integers, whose whole turns fall off its top.  The frequency's rounding is 2^-65 turns
// (or, above 2^-11 turns a token, 2^-53 of itself): below 10^-7 turns at position 2^31.
// Frequencies of half a turn and more lose their whole turns first, the quotient by a turn in two parts (not inlined:
// few models have any, and beside it append of 256 tokens took 10.5 us for 10.2).
static __device__ __noinline__ int64_t turn_per_token_fast(double frequency) {
    constexpr double kPerTurn = 0.15915494309189535, kRest = -9.839338337591243e-18;  // 1 / (2 pi)
    const double turns = frequency * kPerTurn, rest = fma(frequency, kRest, fma(frequency, kPerTurn, -turns));
    return int64_t(uint64_t(__double2ll_rn((turns - floor(turns + 0.5)) * 0x1p64)) + uint64_t(__double2ll_rn(rest * 0x1p64)));
}
__device__ __forceinline__ int64_t turn_per_token(double frequency) {
    if (fabs(frequency) >= 3.14159265) return turn_per_token_fast(frequency);
    return __double2ll_rn(frequency * (18446744073709551616.0 / 6.283185307179586476925));
}
__device__ __forceinline__ int64_t phase_of(int64_t position, double frequency) {
    return int64_t(uint64_t(position) * uint64_t(turn_per_token(frequency)));
}

__device__ __forceinline__ int64_t position_at(const void *positions, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(positions)[i] : int64_t(static_cast<const int32_t *>(positions)[i]);
}

// A tile: 16 tokens of one kv head (see the C header for what lies where).
constexpr int kTile = 16, kGroup = 64;

template <int D>
struct KvTile {
    static constexpr int kGroups = D / kGroup;
    static constexpr int kBytes = 18 * D;
    static constexpr int kKeyPairs = 8 * D, kValues = 9 * D, kValuePairs = 17 * D;
    static constexpr int kBlockGroups = kGroups < 2 ? 1 : 2;  // groups of a block of key words
    static constexpr int kBlockRow = 32 * kBlockGroups;       // bytes of its row

    __host__ __device__ static constexpr int row(int token) { return (token & 8) | ((token & 3) << 1) | ((token >> 2) & 1); }
    // Bytes of the word with channels 8 i + 0..7 of a group, and of the pair.
    __device__ static int key_word(int token, int group, int i) {
        return (group / kBlockGroups) * kTile * kBlockRow + row(token) * kBlockRow +
               4 * (2 * kBlockGroups * (i >> 1) + 2 * (group % kBlockGroups) + (i & 1));
    }
    __device__ static int value_word(int token, int group, int i) {
        const int w = kGroups * i + group;
        return kValues + (w >> 3) * kTile * 32 + token * 32 + (w & 7) * 4;
    }
    __device__ static int pair(bool values, int token, int group) {
        return (values ? kValuePairs : kKeyPairs) + (row(token) * kGroups + group) * 4;
    }
};

// (x & mask) | bits in one instruction; written in C it took two (454 -> 392 instructions a tile of attention,
// 256 requests 468 -> 409 us).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
    return r;
}

// Byte offset of the tile of one head that position p lies in, or -1.
__device__ __forceinline__ int64_t tile_at(const int32_t *table, int width, int64_t num_pages, int64_t p, int page_size, int heads,
                                           int head, int tile_bytes, int32_t *status) {
    if (p < 0) return -1;
    const int64_t index = p / page_size;
    if (index >= width) {
        flag(status, SQ_STATUS_SLOT_RANGE);
        return -1;
    }
    const int page = table[index];
    if (page >= num_pages) {
        flag(status, SQ_STATUS_SLOT_RANGE);
        return -1;
    }
    if (page <= 0) return -1;
    const int tiles = page_size / kTile;
    return ((int64_t(page) * heads + head) * tiles + int(p % page_size) / kTile) * tile_bytes;
}

}  // namespace sq
