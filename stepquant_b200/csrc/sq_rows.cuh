// Sequences of concatenated prompts and state rows of requests, shared by the
// convolution and the scan.
#pragma once

#include "sq_common.cuh"

namespace sq {

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
