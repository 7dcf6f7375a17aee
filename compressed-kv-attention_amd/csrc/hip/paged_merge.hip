// Joins the partial states of the paged attention kernels, and picks their
// instantiation.
#include "paged_attention.h"

#include <algorithm>

namespace kvexp_dev {
namespace paged {
namespace {

// Joins the states of a row: maximum, then the weighted sums. W waves per row,
// wave w the splits w, w + W, ..; lane i takes the weight of its wave's i-th
// split of a batch of 64, then every lane its channels of the batch's rows, in
// split order (the same sum every time). Every row's sums are read, four in
// flight: a split that saw nothing of the row has weight 0 and sums 0.
struct Joined {
    float m = -__builtin_inff(), l = 0.0f;
    float acc[4] = {0, 0, 0, 0};
};

__device__ __forceinline__ float wave_max_all(float x) {
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum_all(float x) {
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

template <int CH> // channels per lane
__device__ __forceinline__ void join_rows(Joined &j, const float *acc, int64_t step, int cnt, float w, int dim) {
    const int lane = lane_id();
#pragma unroll 8
    for (int i = 0; i < cnt; ++i) {
        const float wi = readlane_f32(w, i);
        const float *row = acc + i * step;
#pragma unroll
        for (int k = 0; k < CH; ++k) j.acc[k] = __builtin_fmaf(wi, row[min(lane + kWave * k, dim - 1)], j.acc[k]);
    }
}

// Splits first, first + every, .. below n of the row whose split 0 is in `slot`.
__device__ __forceinline__ void join(Joined &j, const float *acc, const float *ml, int64_t slot, int64_t step, int first,
                                     int every, int n, int dim) {
    const int lane = lane_id(), mine = first < n ? (n - first + every - 1) / every : 0;
    for (int s0 = 0; s0 < mine; s0 += kWave) {
        const int cnt = min(kWave, mine - s0);
        float m = -__builtin_inff(), l = 0.0f;
        if (lane < cnt) {
            const float2 x = *reinterpret_cast<const float2 *>(ml + 2 * (slot + (first + (s0 + lane) * every) * step));
            m = x.x;
            l = x.y;
        }
        const float mn = fmaxf(j.m, wave_max_all(l == 0.0f ? -__builtin_inff() : m));
        const float base = mn == -__builtin_inff() ? 0.0f : mn;
        const float old = exp2_f32(j.m - base), w = l == 0.0f ? 0.0f : exp2_f32(m - base);
        j.m = mn;
        j.l = j.l * old + wave_sum_all(l == 0.0f ? 0.0f : w * l);
#pragma unroll
        for (int k = 0; k < 4; ++k) j.acc[k] *= old;
        const float *rows = acc + (slot + int64_t(first + s0 * every) * step) * dim;
        if (dim <= 64) join_rows<1>(j, rows, every * step * dim, cnt, w, dim);
        else if (dim <= 128) join_rows<2>(j, rows, every * step * dim, cnt, w, dim);
        else join_rows<4>(j, rows, every * step * dim, cnt, w, dim);
    }
}

// Fills in a shared prefix's segments (the host left each one's tensor in
// n_esc and its block in mode): the block's payload and header fields, and the
// records of the segment's rows (a block's records ascend by element).
__global__ __launch_bounds__(256) void prefix_segs_kernel(PrefixSeg *__restrict__ segs, int n,
                                                          const EscJob *__restrict__ jobs) {
    const int i = int(blockIdx.x) * 256 + int(threadIdx.x);
    if (i >= n) return;
    PrefixSeg s = segs[i];
    const EscJob j = jobs[s.n_esc];
    const int b = s.mode;
    const uint8_t *p = j.blob + j.offs[b];
    const BlockHdr h = read_hdr(p);
    const uint32_t *rec = j.pos + j.esc0[b];
    const int n_rec = j.esc0[b + 1] - j.esc0[b];
    auto below = [&](int e) { // records of elements below e
        int lo = 0, hi = n_rec;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (int(rec[mid] & 0xFFFFu) < e) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    const int r0 = below(s.row0 * j.dim), r1 = below((s.row0 + s.rows) * j.dim);
    s.data = p + 8;
    s.esc = rec + r0;
    s.n_esc = max(r1 - r0, 0);
    s.mode = h.mode;
    s.n_tokens = h.n_tokens;
    segs[i] = s;
}

template <bool HALF, int W>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
    __shared__ float part[4][kMaxDim + 2];
    const int hq_all = a.n_kv * a.group;
    const int wave = int(threadIdx.x) >> 6, lane = lane_id();
    const int64_t at = W == 4 ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * 4 + wave;
    if (at >= int64_t(a.batch.n_tokens) * hq_all) return;
    const int tok = int(at / hq_all), hq = int(at - int64_t(tok) * hq_all);
    const int seq = seq_of_wave(a.batch, tok);
    if (seq < 0) return; // a row behind the last sequence
    Rows r;
    find_rows(a, seq, 1, 1, 1, r); // (split and tile 1: no errors raised here)
    const int i = tok - r.first;
    if (i < 0 || i >= r.n) return;
    const int head = hq / a.group, g = hq - head * a.group;
    const int first = W == 4 ? wave : 0;
    Joined j;
    if (a.s_splits > 0) {
        const int len = split_tokens(a.s_len, a.s_splits, a.s_min_split);
        const int n = max(1, (a.s_len + len - 1) / len);
        join(j, a.s_acc, a.s_ml, int64_t(head) * a.s_splits * a.s_rows + int64_t(tok) * a.group + g, a.s_rows, first, W, n, a.dim);
    }
    const int n = max(1, (r.len + r.split_len - 1) / r.split_len);
    join(j, a.acc, a.ml, state_slot(a, r, head, 0, i * a.group + g), a.max_rows, first, W, n, a.dim);
    if constexpr (W == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) part[wave][lane + kWave * k] = j.acc[k];
        if (lane == 0) {
            part[wave][kMaxDim] = j.m;
            part[wave][kMaxDim + 1] = j.l;
        }
        __syncthreads();
        if (wave != 0) return;
        float M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, part[w][kMaxDim]);
        const float base = M == -__builtin_inff() ? 0.0f : M;
        j = Joined{};
        j.m = M;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float l = part[w][kMaxDim + 1], e = l == 0.0f ? 0.0f : exp2_f32(part[w][kMaxDim] - base);
            j.l += l == 0.0f ? 0.0f : e * l;
#pragma unroll
            for (int k = 0; k < 4; ++k) j.acc[k] = __builtin_fmaf(e, part[w][lane + kWave * k], j.acc[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int d = lane + kWave * k;
        if (d < a.dim) a.out.p[int64_t(tok) * a.out.token + int64_t(hq) * a.out.head + d] = to_16<HALF>(finish(j.acc[k], j.l));
    }
    if (lane == 0 && a.lse != nullptr) a.lse[at] = log_sum(j.m, j.l);
}

} // namespace
} // namespace paged
} // namespace kvexp_dev

namespace kvexp_launch {

using namespace kvexp_dev;

#define KVEXP_PAGED_DECL(DP)                                                                       \
    hipError_t paged_few_d##DP(const PagedAttnArgs &a, bool half, bool two, int n_seqs, hipStream_t s); \
    hipError_t paged_many_d##DP(const PagedAttnArgs &a, bool half, int tile_rows, int n_seqs, hipStream_t s);
KVEXP_PAGED_DECL(32)
KVEXP_PAGED_DECL(64)
KVEXP_PAGED_DECL(96)
KVEXP_PAGED_DECL(128)
KVEXP_PAGED_DECL(192)
KVEXP_PAGED_DECL(256)

// tile_rows: 16 or 32 (the few-row kernel), 128 or 256 (the many-row kernel).
hipError_t paged_attention(const PagedAttnArgs &a, bool half, int tile_rows, int n_seqs, hipStream_t s) {
    const bool many = tile_rows > 32, two = tile_rows == 32;
#define KVEXP_PAGED_PICK(DP) \
    if (a.dim <= DP) return many ? paged_many_d##DP(a, half, tile_rows, n_seqs, s) : paged_few_d##DP(a, half, two, n_seqs, s);
    KVEXP_PAGED_PICK(32)
    KVEXP_PAGED_PICK(64)
    KVEXP_PAGED_PICK(96)
    KVEXP_PAGED_PICK(128)
    KVEXP_PAGED_PICK(192)
    KVEXP_PAGED_PICK(256)
    return hipErrorInvalidValue;
}

hipError_t prefix_segs(PrefixSeg *segs, int n, const EscJob *jobs, hipStream_t s) {
    hipLaunchKernelGGL(paged::prefix_segs_kernel, dim3(unsigned((n + 255) / 256)), dim3(256), 0, s, segs, n, jobs);
    return hipGetLastError();
}

hipError_t paged_merge(const PagedAttnArgs &a, bool half, hipStream_t s) {
    const int64_t n = int64_t(a.batch.n_tokens) * a.n_kv * a.group;
    // four waves per row where there are splits for them and their workgroups
    // all run at once (2,048 rows of 32 + 2 splits of 128 channels: 11.3 us, with
    // one wave 14.5; 3,584 rows of 18 + 1 of 64: 15.0 and 10.9)
    const bool four = n <= 2048 && a.n_splits + a.s_splits >= 8;
    auto run = [&](auto kernel, int64_t groups) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(groups)), dim3(256), 0, s, a);
    };
    if (four) half ? run(paged::paged_merge_kernel<true, 4>, n) : run(paged::paged_merge_kernel<false, 4>, n);
    else half ? run(paged::paged_merge_kernel<true, 1>, (n + 3) / 4) : run(paged::paged_merge_kernel<false, 1>, (n + 3) / 4);
    return hipGetLastError();
}

} // namespace kvexp_launch
