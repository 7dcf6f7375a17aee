// Rotary positions and the append to a paged cache with the rotation on the
// way.
//
// A token's pair of channels (x1, x2) of frequency i turns by the angle
// pos[axis(i)] * freq[i]: y1 = (x1 cos - x2 sin) s, y2 = (x2 cos + x1 sin) s.
// Pairs are channels (i, i + n_freq), or (2 i, 2 i + 1); channels past
// 2 n_freq are copied. The gradient is the rotation back (sign -1).
//
// A workgroup takes a few tokens: first the cosines and sines of their
// frequencies to LDS (once per token, for all heads), and each token's place
// in the pages; then the heads, 16 bytes of each half of a pair run per
// thread (general_kernel: one pair per thread, for counts of frequencies that
// are no multiple of 8). The angle is formed in 64 bits as turns
// (pos * freq / 2 pi) and reduced there, so that far positions lose nothing:
// the part of a turn that is left is rounded to 32 bits (an angle error of at
// most pi 2^-24). The products are 32-bit and the result is rounded once.
#include "paged_device.h"

#include <algorithm>
#include <hip/hip_fp16.h>

namespace kvexp_dev {
namespace paged {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 16; // most tokens per workgroup

// The cosine and sine tables are sized at launch: [tokens][n_freq].
extern __shared__ float2 rot_table[];

template <bool HALF>
__device__ __forceinline__ float to_f32(uint32_t b) {
    if constexpr (HALF) return __half2float(__ushort_as_half(uint16_t(b)));
    else return bf16_f32(b);
}
template <bool HALF>
__device__ __forceinline__ uint32_t from_f32(float x) {
    if constexpr (HALF) return __half_as_ushort(__float2half_rn(x));
    else return uint32_t(__builtin_bit_cast(uint16_t, __bf16(x)));
}

struct RotPlace {
    int64_t k, v; // element offsets of head 0 in the pools; k < 0: not written
};

__device__ __forceinline__ int64_t position(const RopeDev &r, int axis, int t, int64_t place) {
    if (r.pos == nullptr) return place + r.offset;
    const int64_t at = int64_t(axis) * r.axis_stride + t;
    return r.pos64 ? static_cast<const int64_t *>(r.pos)[at] : int64_t(static_cast<const int32_t *>(r.pos)[at]);
}

// The token's place: its sequence's next index and row in the pages.
__device__ __forceinline__ RotPlace place_of(const RotateArgs &a, int t, int64_t &index, bool &held) {
    RotPlace r{-1, 0};
    index = t;
    held = true;
    if (a.n_kv == 0) return r;
    const BatchDev &b = a.batch;
    const int seq = seq_of(b, t);
    held = seq >= 0;
    index = 0;
    if (!held) return r;
    int first, n;
    new_rows(b, seq, first, n);
    const int at = b.lens[seq] - n + (t - first);
    index = at;
    if (at < 0) return r; // the sequence is shorter than its new tokens
    const int64_t col = page_of(a.pool, at);
    if (col >= b.table_width) {
        atomicOr(a.status, kStLength);
        return r;
    }
    const int page = b.table[int64_t(seq) * b.table_stride + col];
    if (uint32_t(page) >= uint32_t(a.pool.n_pages)) {
        atomicOr(a.status, kStPage);
        return r;
    }
    const int64_t row = at - col * a.pool.page_tokens;
    r.k = int64_t(page) * a.pool.k_page + row * a.pool.k_token;
    r.v = int64_t(page) * a.pool.v_page + row * a.pool.v_token;
    return r;
}

// Cosines, sines and places of the group's tokens.
__device__ __forceinline__ void fill_tables(const RotateArgs &a, int t0, int nt, RotPlace *places, int64_t *index,
                                            int *held) {
    const int tid = int(threadIdx.x);
    if (tid < nt) {
        bool h;
        places[tid] = place_of(a, t0 + tid, index[tid], h);
        held[tid] = h;
    }
    if (a.rope.pos == nullptr) __syncthreads(); // the angles need the indexes
    const int nf = a.rope.n_freq;
    for (int i = tid; i < nt * nf; i += kRotThreads) {
        const int tt = i / nf, f = i - tt * nf;
        const int axis = a.rope.axes != nullptr ? min(int(a.rope.axes[f]), a.rope.n_axes - 1) : 0;
        const int64_t pos = position(a.rope, axis, t0 + tt, a.rope.pos == nullptr ? index[tt] : 0);
        const double turns = double(pos) * double(a.rope.freq[f]) * 0.15915494309189533577;
        const float part = float(turns - __builtin_rint(turns)) * 2.0f; // half turns in [-1, 1]
        float s, c;
        sincospif(part, &s, &c);
        rot_table[i] = make_float2(c * a.rope.scale, s * a.rope.scale * a.rope.sign);
    }
    __syncthreads();
}

typedef uint32_t rot_u32x4 __attribute__((ext_vector_type(4)));

template <bool HALF>
__device__ __forceinline__ void unpack8(const rot_u32x4 &x, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = to_f32<HALF>(x[i] & 0xFFFFu);
        f[2 * i + 1] = to_f32<HALF>(x[i] >> 16);
    }
}
template <bool HALF>
__device__ __forceinline__ rot_u32x4 pack8(const float (&f)[8]) {
    rot_u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = from_f32<HALF>(f[2 * i]) | (from_f32<HALF>(f[2 * i + 1]) << 16);
    return x;
}

// Source and destination of head hh of token slot tt (heads: the queries, the
// keys, the values); false: nothing to write.
__device__ __forceinline__ bool head_rows(const RotateArgs &a, int t, int hh, const RotPlace &pl, bool held,
                                          const uint16_t *&src, uint16_t *&dst, bool &rotate) {
    rotate = true;
    if (hh < a.n_q) {
        src = a.q.p + int64_t(t) * a.q.token + int64_t(hh) * a.q.head;
        dst = a.q_out.p + int64_t(t) * a.q_out.token + int64_t(hh) * a.q_out.head;
        return held;
    }
    hh -= a.n_q;
    if (hh < a.n_kv) {
        src = a.k.p + int64_t(t) * a.k.token + int64_t(hh) * a.k.head;
        dst = a.pool.k + pl.k + int64_t(hh) * a.pool.k_head;
        return pl.k >= 0;
    }
    hh -= a.n_kv;
    rotate = false;
    src = a.v.p + int64_t(t) * a.v.token + int64_t(hh) * a.v.head;
    dst = a.pool.v + pl.v + int64_t(hh) * a.pool.v_head;
    return pl.k >= 0;
}

template <bool HALF, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotate_kernel(RotateArgs a) {
    __shared__ RotPlace places[kRotTokens];
    __shared__ int64_t index[kRotTokens];
    __shared__ int held[kRotTokens];
    const int t0 = int(blockIdx.x) * a.tokens_per_group;
    const int nt = min(a.tokens_per_group, a.n_tokens - t0);
    fill_tables(a, t0, nt, places, index, held);
    const int nf = a.rope.n_freq;
    // a rotated head: its pair runs, then 8 channels per unit; a copied one: 8 channels per unit
    const int pairs = INTERLEAVED ? nf / 4 : nf / 8;
    const int up = pairs + (a.dim - 2 * nf) / 8, uv = a.dim / 8;
    const int rot_units = (a.n_q + a.n_kv) * up, units = rot_units + a.n_kv * uv;
    for (int i = int(threadIdx.x); i < nt * units; i += kRotThreads) {
        const int tt = i / units, u = i - tt * units;
        int hh, c;
        if (u < rot_units) {
            hh = u / up;
            c = u - hh * up;
        } else {
            const int w = u - rot_units;
            hh = w / uv;
            c = w - hh * uv;
            hh += a.n_q + a.n_kv;
        }
        const uint16_t *src;
        uint16_t *dst;
        bool rot;
        if (!head_rows(a, t0 + tt, hh, places[tt], held[tt] != 0, src, dst, rot)) continue;
        if (!rot || c >= pairs) { // copied channels
            const int ch = rot ? 2 * nf + 8 * (c - pairs) : 8 * c;
            *reinterpret_cast<rot_u32x4 *>(dst + ch) = *reinterpret_cast<const rot_u32x4 *>(src + ch);
            continue;
        }
        float x[8];
        if constexpr (INTERLEAVED) {
            unpack8<HALF>(*reinterpret_cast<const rot_u32x4 *>(src + 8 * c), x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 cs = rot_table[tt * nf + 4 * c + k];
                const float p = x[2 * k], q = x[2 * k + 1];
                x[2 * k] = __builtin_fmaf(p, cs.x, -(q * cs.y));
                x[2 * k + 1] = __builtin_fmaf(q, cs.x, p * cs.y);
            }
            *reinterpret_cast<rot_u32x4 *>(dst + 8 * c) = pack8<HALF>(x);
        } else {
            float y[8];
            unpack8<HALF>(*reinterpret_cast<const rot_u32x4 *>(src + 8 * c), x);
            unpack8<HALF>(*reinterpret_cast<const rot_u32x4 *>(src + nf + 8 * c), y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 cs = rot_table[tt * nf + 8 * c + k];
                const float p = x[k], q = y[k];
                x[k] = __builtin_fmaf(p, cs.x, -(q * cs.y));
                y[k] = __builtin_fmaf(q, cs.x, p * cs.y);
            }
            *reinterpret_cast<rot_u32x4 *>(dst + 8 * c) = pack8<HALF>(x);
            *reinterpret_cast<rot_u32x4 *>(dst + nf + 8 * c) = pack8<HALF>(y);
        }
    }
}

// Any count of frequencies: one pair of channels per thread and step.
template <bool HALF>
__global__ __launch_bounds__(kRotThreads) void rotate_general_kernel(RotateArgs a) {
    __shared__ RotPlace places[kRotTokens];
    __shared__ int64_t index[kRotTokens];
    __shared__ int held[kRotTokens];
    const int t0 = int(blockIdx.x) * a.tokens_per_group;
    const int nt = min(a.tokens_per_group, a.n_tokens - t0);
    fill_tables(a, t0, nt, places, index, held);
    const int nf = a.rope.n_freq, up = a.dim / 2;
    const int units = (a.n_q + 2 * a.n_kv) * up;
    for (int i = int(threadIdx.x); i < nt * units; i += kRotThreads) {
        const int tt = i / units, u = i - tt * units;
        const int hh = u / up, c = u - hh * up;
        const uint16_t *src;
        uint16_t *dst;
        bool rot;
        if (!head_rows(a, t0 + tt, hh, places[tt], held[tt] != 0, src, dst, rot)) continue;
        const bool turn = rot && c < nf;
        const int c1 = !turn || a.rope.interleaved ? 2 * c : c;
        const int c2 = !turn || a.rope.interleaved ? 2 * c + 1 : c + nf;
        const uint32_t x1 = src[c1], x2 = src[c2];
        if (!turn) {
            dst[c1] = uint16_t(x1);
            dst[c2] = uint16_t(x2);
            continue;
        }
        const float2 cs = rot_table[tt * nf + c];
        const float p = to_f32<HALF>(x1), q = to_f32<HALF>(x2);
        dst[c1] = uint16_t(from_f32<HALF>(__builtin_fmaf(p, cs.x, -(q * cs.y))));
        dst[c2] = uint16_t(from_f32<HALF>(__builtin_fmaf(q, cs.x, p * cs.y)));
    }
}

} // namespace
} // namespace paged
} // namespace kvexp_dev

namespace kvexp_launch {

using namespace kvexp_dev;

// `a` but for tokens_per_group, which is chosen here.
hipError_t rotate(RotateArgs a, bool half, hipStream_t s) {
    using namespace kvexp_dev::paged;
    if (a.n_tokens <= 0) return hipSuccess;
    // Four tokens per workgroup once there are workgroups for every CU (32,760
    // tokens x 12 heads x 128 channels: 38 us; one token 55, two 46, eight 41,
    // sixteen 48, whose one round of workgroups makes its tables all at once
    // and then streams), more where four are less than a unit per thread
    // (200,000 tokens of one head of 64 channels: 23 us, with four tokens 44).
    const int64_t units = (int64_t(a.n_q) + 2 * a.n_kv) * a.dim / 16; // (about)
    a.tokens_per_group = std::max(1, std::min(4, a.n_tokens / 2048));
    while (2 * a.tokens_per_group <= kRotTokens && a.tokens_per_group * units < kRotThreads &&
           a.n_tokens / (2 * a.tokens_per_group) >= 2048)
        a.tokens_per_group *= 2;
    const unsigned groups = unsigned((a.n_tokens + a.tokens_per_group - 1) / a.tokens_per_group);
    const size_t lds = size_t(a.tokens_per_group) * size_t(std::max(1, a.rope.n_freq)) * sizeof(float2);
    const int nf = a.rope.n_freq;
    const bool wide = a.rope.interleaved ? nf % 4 == 0 : nf % 8 == 0;
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(groups), dim3(kRotThreads), lds, s, a); };
    if (!wide) half ? run(rotate_general_kernel<true>) : run(rotate_general_kernel<false>);
    else if (a.rope.interleaved) half ? run(rotate_kernel<true, true>) : run(rotate_kernel<false, true>);
    else half ? run(rotate_kernel<true, false>) : run(rotate_kernel<false, false>);
    return hipGetLastError();
}

} // namespace kvexp_launch
