// Sequences of concatenated prompts and state rows of requests, shared by the
// convolution and the scan.
#pragma once

#include "sq_common.cuh"

namespace sq {

// A strip, a chunk's tile or a batch of tokens may begin anywhere before the last token, and its end
// is an int too.
constexpr int kMostTokens = 0x7fff0000;

// Token range of sequence n, clamped to [0, tokens).
__device__ __forceinline__ int2 sequence_range(const int32_t *cu, int n, int tokens) {
    const int b = max(0, min(cu[n], tokens));
    return make_int2(b, max(b, min(cu[n + 1], tokens)));
}

// Strips of `strip` tokens of the concatenated sequences: sequence n owns the
// indices from cu[n] / strip + n on, at least as many as its strips (and one if
// it is empty), so a CTA finds its sequence by bisection from the ends alone and
// the host knows their number, tokens / strip + sequences.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int seqs, int tokens, int strip, int64_t index) {
    int lo = 0, hi = seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (max(0, min(cu[mid], tokens)) / strip + int64_t(mid) <= index) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Zeros into the rows of y (contiguous, `row` bytes each, an even number) that no sequence owns:
// those before the first one's and past the last one's, by the threads of CTAs 0 .. ctas - 1.
// Not inlined: beside it the schedule of the kernel around gets worse (convolution of 32768 x 8192
// in 187 us for 180).
__device__ __noinline__ static void clear_outside(void *y, int64_t row, const int32_t *cu, int seqs, int tokens, unsigned cta,
                                                  unsigned ctas) {
    const int64_t index = int64_t(cta) * blockDim.x + threadIdx.x, step = int64_t(ctas) * blockDim.x;
    const int begin = sequence_range(cu, 0, tokens).x, end = sequence_range(cu, seqs - 1, tokens).y;
    auto clear = [&](uintptr_t from, uintptr_t to) {
        const uintptr_t low = min((from + 15) & ~uintptr_t(15), to), high = max(low, to & ~uintptr_t(15));
        for (uintptr_t p = from + 2 * index; p < low; p += 2 * step) *reinterpret_cast<uint16_t *>(p) = 0;
        for (uintptr_t p = low + 16 * index; p < high; p += 16 * step) *reinterpret_cast<uint4 *>(p) = make_uint4(0, 0, 0, 0);
        for (uintptr_t p = high + 2 * index; p < to; p += 2 * step) *reinterpret_cast<uint16_t *>(p) = 0;
    };
    const uintptr_t base = reinterpret_cast<uintptr_t>(y);
    clear(base, base + begin * row);
    clear(base + end * row, base + tokens * row);
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

}  // namespace sq
