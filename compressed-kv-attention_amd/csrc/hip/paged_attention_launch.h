// Launches of the paged attention kernels at one channel count (one
// instantiation unit each).
#pragma once
#include "paged_attention.h"

#define KVEXP_PAGED_LAUNCH(DP)                                                                                        \
    hipError_t paged_few_d##DP(const kvexp_dev::PagedAttnArgs &a, bool half, int n_seqs, hipStream_t s) {             \
        using namespace kvexp_dev::paged;                                                                             \
        const dim3 grid(unsigned(a.n_splits), unsigned(a.n_kv * a.row_tiles), unsigned(n_seqs));                      \
        if (half) hipLaunchKernelGGL((paged_few_kernel<DP, true>), grid, dim3(kPagedThreads), 0, s, a);               \
        else hipLaunchKernelGGL((paged_few_kernel<DP, false>), grid, dim3(kPagedThreads), 0, s, a);                   \
        return hipGetLastError();                                                                                     \
    }                                                                                                                 \
    hipError_t paged_many_d##DP(const kvexp_dev::PagedAttnArgs &a, bool half, int n_seqs, hipStream_t s) {            \
        using namespace kvexp_dev::paged;                                                                             \
        const dim3 grid(unsigned(a.n_splits), unsigned(a.n_kv * a.row_tiles), unsigned(n_seqs));                      \
        if (a.px != nullptr) hipLaunchKernelGGL((paged_many_kernel<DP, false, 1>), grid, dim3(kPagedThreads), 0, s, a); \
        else if (half) hipLaunchKernelGGL((paged_many_kernel<DP, true, 0>), grid, dim3(kPagedThreads), 0, s, a);      \
        else hipLaunchKernelGGL((paged_many_kernel<DP, false, 0>), grid, dim3(kPagedThreads), 0, s, a);               \
        return hipGetLastError();                                                                                     \
    }
