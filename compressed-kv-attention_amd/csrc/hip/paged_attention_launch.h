// Launches of the paged attention kernels at one channel count (one
// instantiation unit each).
#pragma once
#include "paged_attention.h"

namespace kvexp_dev {
namespace paged {

inline dim3 attention_grid(const PagedAttnArgs &a, int n_seqs) {
    return dim3(unsigned(a.n_splits) * unsigned(a.n_kv) * unsigned(a.row_tiles) * unsigned(n_seqs));
}

template <int DP, bool HALF, int NC, bool HALVES>
void launch_few_c(const PagedAttnArgs &a, int n_seqs, hipStream_t s) {
    const dim3 grid = attention_grid(a, n_seqs);
    // rows of several new tokens see different tokens
    if (!a.shared && a.batch.max_new > 1)
        hipLaunchKernelGGL((paged_few_kernel<DP, HALF, NC, HALVES, true>), grid, dim3(kPagedThreads), 0, s, a);
    else hipLaunchKernelGGL((paged_few_kernel<DP, HALF, NC, HALVES, false>), grid, dim3(kPagedThreads), 0, s, a);
}

template <int DP, bool HALF>
void launch_few(const PagedAttnArgs &a, bool two, int n_seqs, hipStream_t s) {
    const bool halves = a.pool.page_tokens % 16 == 0;
    if constexpr (kFewRowsAt<DP> == 32)
        if (two) return halves ? launch_few_c<DP, HALF, 2, true>(a, n_seqs, s) : launch_few_c<DP, HALF, 2, false>(a, n_seqs, s);
    halves ? launch_few_c<DP, HALF, 1, true>(a, n_seqs, s) : launch_few_c<DP, HALF, 1, false>(a, n_seqs, s);
}

template <int DP, bool HALF, int SRC, int NW>
hipError_t launch_many_waves(const PagedAttnArgs &a, int n_seqs, hipStream_t s) {
    // (past the default 64 KiB of LDS; the attribute is a device's own, so every call sets it)
    constexpr size_t lds = sizeof(ManyLds<DP, SRC, NW>);
    if (lds > 64 * 1024) {
        const hipError_t set =
            hipFuncSetAttribute(reinterpret_cast<const void *>(paged_many_kernel<DP, HALF, SRC, NW>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (set != hipSuccess) return set;
    }
    hipLaunchKernelGGL((paged_many_kernel<DP, HALF, SRC, NW>), attention_grid(a, n_seqs), dim3(64 * NW),
                       lds, s, a);
    return hipGetLastError();
}

template <int DP, bool HALF, int SRC>
hipError_t launch_many_src(const PagedAttnArgs &a, int tile_rows, int n_seqs, hipStream_t s) {
    if constexpr (many_rows(DP, SRC == 1) == 256)
        if (tile_rows == 256) return launch_many_waves<DP, HALF, SRC, 8>(a, n_seqs, s);
    return launch_many_waves<DP, HALF, SRC, 4>(a, n_seqs, s);
}

template <int DP>
hipError_t launch_many(const PagedAttnArgs &a, bool half, int tile_rows, int n_seqs, hipStream_t s) {
    if (a.px != nullptr) return launch_many_src<DP, false, 1>(a, tile_rows, n_seqs, s);
    return half ? launch_many_src<DP, true, 0>(a, tile_rows, n_seqs, s) : launch_many_src<DP, false, 0>(a, tile_rows, n_seqs, s);
}

} // namespace paged
} // namespace kvexp_dev

#define KVEXP_PAGED_LAUNCH(DP)                                                                                        \
    hipError_t paged_few_d##DP(const kvexp_dev::PagedAttnArgs &a, bool half, bool two, int n_seqs, hipStream_t s) {   \
        if (half) kvexp_dev::paged::launch_few<DP, true>(a, two, n_seqs, s);                                          \
        else kvexp_dev::paged::launch_few<DP, false>(a, two, n_seqs, s);                                              \
        return hipGetLastError();                                                                                     \
    }                                                                                                                 \
    hipError_t paged_many_d##DP(const kvexp_dev::PagedAttnArgs &a, bool half, int tile_rows, int n_seqs,         \
                                 hipStream_t s) {                                                                     \
        return kvexp_dev::paged::launch_many<DP>(a, half, tile_rows, n_seqs, s);                                      \
    }
