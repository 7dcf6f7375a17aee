// Device helpers of the paged-cache kernels.
#pragma once

#include "kvexp_device.h"
#include "paged_types.h"

namespace kvexp_dev {
namespace paged {

// t / page_tokens for 0 <= t < 2^31: a multiplication (the host finds magic
// and shift so that the quotient is exact), or a shift for powers of two.
__device__ __forceinline__ int page_of(const PoolDev &p, int t) {
    if (p.page_magic == 0) return t >> p.page_shift;
    return int((uint64_t(uint32_t(t)) * p.page_magic) >> (32 + p.page_shift));
}

// First row and count of sequence b's new tokens, held to the call's rows.
__device__ __forceinline__ void new_rows(const BatchDev &b, int seq, int &first, int &n) {
    if (b.starts == nullptr) {
        first = seq * b.n_new;
        n = b.n_new;
        return;
    }
    const int s0 = b.starts[seq], s1 = b.starts[seq + 1];
    first = min(max(s0, 0), b.n_tokens);
    n = max(min(s1, b.n_tokens) - first, 0);
}

// The sequence of row t: the last b with starts[b] <= t (-1: none, or rows
// behind the last sequence).
__device__ __forceinline__ int seq_of(const BatchDev &b, int t) {
    if (b.starts == nullptr) return t / b.n_new;
    int lo = 0, hi = b.n_seqs; // starts[lo] <= t < starts[hi], if any
    if (t < b.starts[0] || t >= b.starts[b.n_seqs]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same by a whole wave, for a t that its lanes share: 64 starts at a time.
__device__ __forceinline__ int seq_of_wave(const BatchDev &b, int t) {
    if (b.starts == nullptr) return t / b.n_new;
    if (t < b.starts[0] || t >= b.starts[b.n_seqs]) return -1;
    int lo = 0, hi = b.n_seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + kWave - 1) / kWave;
        const int64_t at = int64_t(lo) + int64_t(lane_id()) * step;
        const uint64_t below = __ballot(at < hi && b.starts[at] <= t);
        lo += max(__popcll(below) - 1, 0) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

} // namespace paged
} // namespace kvexp_dev
