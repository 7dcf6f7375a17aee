// Attention over a paged cache and over a prefix that a batch shares
// (templates; instantiated per head_dim in paged_attention_d*.hip).
//
// A query row r of a (sequence, KV head) sees the tokens [0, limit_r). With
// s_j = scale2 * (q . k_j) (scale2 = scale log2 e), m the running maximum and
// p_j = 2^(s_j - m), a pass over the tokens keeps m, l = sum p_j and
// acc = sum p_j v_j, and turns acc and l by 2^(m_old - m) when m moves. A
// token range per workgroup; the states of a row's ranges are joined by
// paged_merge_kernel: M = max m_i, out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i,
// lse = (M + log2 l) ln 2. A row that sees nothing gives 0 and -inf.
//
// Both kernels form S^T = K Q^T and O^T = V^T P^T on the matrix cores, so that
// a query row is a column of both products: a lane holds its row's scores, its
// maximum, and its outputs, and P goes from the first product's result to the
// second's operand without a move (the tokens of a lane's results are taken as
// the tokens of its operand; V is read in the same order).
#pragma once

#include "attention_team.h"
#include "paged_device.h"

#include <type_traits>

#include <hip/hip_fp16.h>

namespace kvexp_dev {
namespace paged {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = 4;

template <bool HALF>
__device__ __forceinline__ f32x4 mfma16(const u32x4a &a, const u32x4a &b, const f32x4 &c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool HALF>
__device__ __forceinline__ f32x16 mfma32(const u32x4a &a, const u32x4a &b, const f32x16 &c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two floats to 16 bits each, rounded to nearest, x in the low half.
template <bool HALF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (HALF) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{_Float16(x), _Float16(y)});
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{__bf16(x), __bf16(y)});
    }
}
template <bool HALF>
__device__ __forceinline__ float low_f32(uint32_t w) {
    if constexpr (HALF) return __half2float(__ushort_as_half(uint16_t(w & 0xFFFFu)));
    else return bits_f32(w << 16);
}
template <bool HALF>
__device__ __forceinline__ float high_f32(uint32_t w) {
    if constexpr (HALF) return __half2float(__ushort_as_half(uint16_t(w >> 16)));
    else return bits_f32(w & 0xFFFF0000u);
}
template <bool HALF>
__device__ __forceinline__ uint16_t to_16(float x) {
    return uint16_t(pack2<HALF>(x, 0.0f) & 0xFFFFu);
}

__device__ __forceinline__ float exp2_f32(float x) { return __builtin_amdgcn_exp2f(x); }

// Whether either half of a pair of values is an infinity or a NaN.
template <bool HALF>
__device__ __forceinline__ bool wild2(uint32_t w) {
    constexpr uint32_t E = HALF ? 0x7C00u : 0x7F80u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}

// Infinities and NaN among V of tokens that some rows of a tile see and others
// do not: the product with P would carry 0 times them into the rows that do not.
// Such a tile takes its product without them, and a second one, of 1 in their
// places and 1 for the tokens that a row sees, says which outputs they reach:
// those get an infinity of their sign, or NaN (both signs).
template <bool HALF>
struct Wild {
    static constexpr uint32_t E = HALF ? 0x7C00u : 0x7F80u, One = HALF ? 0x3C00u : 0x3F80u;
    // the halves that are finite, the others 0
    static __device__ __forceinline__ uint32_t without(uint32_t w) {
        const uint32_t lo = (w & E) == E ? 0xFFFFu : 0u, hi = (w & (E << 16)) == (E << 16) ? 0xFFFF0000u : 0u;
        return w & ~(lo | hi);
    }
    // 1 where a half reaches plus (or minus) infinity or NaN
    static __device__ __forceinline__ uint32_t only(uint32_t w, bool minus) {
        auto half = [&](uint32_t x) { // plus: all but -inf; minus: all but +inf
            return (x & E) == E && x != (minus ? E : (E | 0x8000u)) ? One : 0u;
        };
        return half(w & 0xFFFFu) | (half(w >> 16) << 16);
    }
    static __device__ __forceinline__ float reach(float z, bool minus) {
        return z > 0.0f ? (minus ? -__builtin_inff() : __builtin_inff()) : 0.0f;
    }
};

// The rows of a workgroup: which query rows, which tokens they see.
struct Rows {
    int seq, head;
    int first;  // first token row of the sequence (or of the call, shared)
    int n;      // its new tokens
    int len;    // tokens that may be seen
    int count;  // rows: n * group
    int t0, t1; // the split's tokens (t1: past the last token any row of the tile sees)
    int split_len;
    bool used;  // the split holds tokens of the sequence
};

// Tokens per split: at least min_split (a multiple of kSplitStep), and n_splits
// of them reach len.
constexpr int kSplitStep = 64;
__device__ __forceinline__ int split_tokens(int len, int n_splits, int min_split) {
    const int even = len / n_splits + (len % n_splits != 0);
    return max(min_split, (even + kSplitStep - 1) / kSplitStep * kSplitStep);
}

// Raises the call's length errors once per sequence.
__device__ __forceinline__ void find_rows(const PagedAttnArgs &a, int seq, int split, int tile, int tile_rows,
                                          Rows &r) {
    r.seq = seq;
    if (a.shared) {
        r.first = 0;
        r.n = a.batch.n_tokens;
        r.len = a.len;
    } else {
        int n;
        new_rows(a.batch, seq, r.first, n);
        r.n = min(n, a.batch.max_new);
        const int held = a.batch.lens[seq];
        const int64_t most = int64_t(a.batch.table_width) * a.pool.page_tokens;
        r.len = int(min(int64_t(max(held, 0)), most));
        if ((n != r.n || held > r.len) && split == 0 && tile == 0 && threadIdx.x == 0) atomicOr(a.status, kStLength);
    }
    r.count = r.n * a.group;
    r.split_len = split_tokens(r.len, a.n_splits, a.min_split);
    r.t0 = min(int64_t(split) * r.split_len, int64_t(r.len));
    r.used = split == 0 || r.t0 < r.len;
    const int last = min((tile + 1) * tile_rows, r.count) - 1; // last row of the tile
    int seen = r.len;
    if (!a.shared) seen = max(0, min(r.len, r.len - r.n + last / a.group + 1));
    r.t1 = min(r.t0 + r.split_len, seen);
}

// What a workgroup works on. Consecutive workgroups go to the eight XCDs in
// turn, so the order decides what shares an XCD and its L2: heads first (they
// have equal work), then row tiles (the last first, which see the most tokens),
// then sequences, turned by the split so that the splits of a long sequence, and
// the first splits, which every sequence has, spread over all of them. (With the
// splits innermost, 32 or 64 of them: every sequence's split 0 on one XCD, and a
// draft step of 16 sequences took 97 and 121 us where 48 splits took 63.)
__device__ __forceinline__ void find_work(const PagedAttnArgs &a, int &split, int &head, int &tile, int &seq) {
    uint32_t w = blockIdx.x;
    const uint32_t seqs = a.shared ? 1u : uint32_t(a.batch.n_seqs);
    head = int(w % uint32_t(a.n_kv));
    w /= uint32_t(a.n_kv);
    tile = a.row_tiles - 1 - int(w % uint32_t(a.row_tiles));
    w /= uint32_t(a.row_tiles);
    split = int(w / seqs);
    seq = int((w % seqs + uint32_t(split)) % seqs);
}

// Tokens that row `row` sees (0 past the rows).
__device__ __forceinline__ int row_limit(const PagedAttnArgs &a, const Rows &r, int row) {
    if (row >= r.count) return 0;
    if (a.shared) return r.len;
    return max(0, min(r.len, r.len - r.n + row / a.group + 1));
}

// Row `row`'s token row in the call's tensors.
__device__ __forceinline__ int row_token(const PagedAttnArgs &a, const Rows &r, int row) {
    return r.first + row / a.group;
}

__device__ __forceinline__ int page_at(const PagedAttnArgs &a, const int32_t *table, int tok, int &in_page) {
    const int col = page_of(a.pool, tok);
    in_page = tok - col * a.pool.page_tokens;
    int page = table[col];
    if (uint32_t(page) >= uint32_t(a.pool.n_pages)) {
        atomicOr(a.status, kStPage);
        page = 0;
    }
    return page;
}

// The state slot of a row and split.
__device__ __forceinline__ int64_t state_slot(const PagedAttnArgs &a, const Rows &r, int head, int split, int row) {
    return (int64_t(head) * a.n_splits + split) * a.max_rows + int64_t(r.first) * a.group + row;
}

// The sums of a row that saw l 0 are nothing: its output is 0.
__device__ __forceinline__ float finish(float acc, float l) { return l == 0.0f ? 0.0f : acc / l; }
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994530942f;
}

// One channel of a row's state, to its slot or, where the call has one split,
// to the output.
template <bool HALF>
__device__ __forceinline__ void write_state(const PagedAttnArgs &a, const Rows &r, int head, int split, int row, int d,
                                            float m, float l, float acc) {
    if (a.direct) {
        const int64_t tok = row_token(a, r, row);
        const int hq = head * a.group + row % a.group;
        a.out.p[tok * a.out.token + int64_t(hq) * a.out.head + d] = to_16<HALF>(finish(acc, l));
        if (d == 0 && a.lse != nullptr) a.lse[tok * (a.n_kv * a.group) + hq] = log_sum(m, l);
        return;
    }
    const int64_t slot = state_slot(a, r, head, split, row);
    a.acc[slot * a.dim + d] = acc;
    if (d == 0) {
        a.ml[2 * slot] = m;
        a.ml[2 * slot + 1] = l;
    }
}

// --------------------------------------------------------------- few rows --
// Up to 16 NC query rows per workgroup (a decode step's queries of one KV head;
// a few draft tokens): 16 x 16 x 32 products, one per 16 tokens and 32
// channels. K and V go from memory to registers, each once: lane (c, g) of a
// product takes 8 channels of token c of K, and of V all its channels (DP / 16
// of them) of the 8 tokens 4 g .. 4 g + 3 and 16 + 4 g .., which its own P
// values belong to; a few byte permutes pair the tokens. The four waves take
// the split's 32-token tiles in turn and join their states at the end in LDS.
//
// Bound: memory. A wave requests its next tile before it works on the one it
// holds, and the pages of the tile after that: in the first form of this loop
// every row's address waited for its own table entry, and ten such round trips
// per tile took 167 us where the loads alone need 60 (64 sequences of 1K to
// 32K tokens, 2 heads x 7 queries of 64 channels). HALVES: pages of a multiple
// of 16 tokens, so that 16 tokens share one entry, which then is a scalar; else
// a lane looks up one token of the tile and the others fetch it from there.
template <int DP>
struct Few {
    static constexpr int KS = DP / 32;   // steps of 32 channels
    static constexpr int C = DP / 16;    // channels of V per lane
    static constexpr int VW = C / 2;     // their dwords
    static constexpr int JC = DP > 192 ? DP / 2 : DP; // channels joined at a time (LDS below 64 KiB)
    static constexpr int Row = JC + 4;   // floats per row of the joint state
    // A second tile in registers, and the waves per SIMD that the registers then
    // allow. More waves hide more than a tile ahead does where both do not fit:
    // four sequences of up to 65,536 tokens, 8 heads x 4 queries of 128 channels,
    // 176 us with a tile ahead (two waves), 129 without (three); at 64 channels
    // both fit three waves (sequences of 1K to 32K: 76 us, 79 with four waves
    // and no tile ahead). Two products of rows at 128 channels: 75 us with one
    // wave, 62 with two (16 sequences of up to 8,192, 32 rows).
    template <int NC>
    static constexpr bool Ahead = DP <= 64 && NC == 1;
    // The next tile's K requested as soon as this one's has given its scores,
    // where the registers hold what that keeps alive (8 queries of 256
    // channels: 87 -> 80 us; at 128 channels it spills, 118 -> 142).
    static constexpr bool Early = DP > 192;
    template <int NC, bool CAUSAL>
    static constexpr int Occ = CAUSAL ? (DP <= 96 || (DP == 128 && NC == 1) ? 2 : 1)
                               : NC > 1 ? 2
                               : DP <= 32 ? 4
                               : DP <= 128 ? 3
                               : DP <= 192 ? 2 : 1;
};

// N dwords at a 4-byte aligned address.
template <int N>
__device__ __forceinline__ void load_words(const uint16_t *p, uint32_t *w) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
    typedef uint32_t x4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t x2 __attribute__((ext_vector_type(2), aligned(4)));
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const x4 v = *reinterpret_cast<const x4 *>(q + i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
    if (N - i >= 2) {
        const x2 v = *reinterpret_cast<const x2 *>(q + i);
        w[i] = v.x, w[i + 1] = v.y;
        i += 2;
    }
    if (N - i == 1) w[i] = q[i];
}

template <int DP>
struct FewTile {
    u32x4a k[2][Few<DP>::KS];
    uint32_t v[8][Few<DP>::VW];
};

// Where a tile's tokens lie. HALVES: page and place of tokens 0 and 16 (the
// same in every lane); else of token lane % 32.
template <bool HALVES>
struct FewPlaces;
template <>
struct FewPlaces<true> {
    int page[2], in_page[2];
};
template <>
struct FewPlaces<false> {
    int page, in_page;
};

// The table entries of the tile from `tok` (tokens past the last read the
// last one's).
template <bool HALVES>
__device__ __forceinline__ void few_places(const PoolDev &pool, const int32_t *table, int tok, int last,
                                           FewPlaces<HALVES> &p) {
    if constexpr (HALVES) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int t = min(tok + 16 * j, last & ~15);
            const int col = page_of(pool, t);
            p.in_page[j] = t - col * pool.page_tokens;
            p.page[j] = table[col];
        }
    } else {
        const int t = min(tok + (lane_id() & 31), last);
        const int col = page_of(pool, t);
        p.in_page = t - col * pool.page_tokens;
        p.page = table[col];
    }
}

// A page number held to the pool; `bad` notes the others.
__device__ __forceinline__ int held_page(const PoolDev &pool, int page, bool &bad) {
    const bool out = uint32_t(page) >= uint32_t(pool.n_pages);
    bad |= out;
    return out ? 0 : page;
}

// Requests K and V of the tile from `tok` (tokens past `last` are read as tokens
// that some row sees; what they give is not used). V false: K, and V otherwise.
template <int DP, bool HALVES, bool V>
__device__ __forceinline__ void few_load(const PagedAttnArgs &a, const uint16_t *base, int tok, int last, int vc,
                                         const FewPlaces<HALVES> &p, bool &bad, FewTile<DP> &f) {
    using F = Few<DP>;
    const int lane = wave::lane_here(), c = lane & 15, g = lane >> 4; // (not held across the loop)
    const int64_t page_step = V ? a.pool.v_page : a.pool.k_page, token_step = V ? a.pool.v_token : a.pool.k_token;
    auto key = [&](const uint16_t *row, int j) {
#pragma unroll
        for (int i = 0; i < F::KS; ++i)
            f.k[j][i] = *reinterpret_cast<const u32x4a *>(row + min(32 * i + 8 * g, a.dim - 8));
    };
    if constexpr (HALVES) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int page = held_page(a.pool, __builtin_amdgcn_readfirstlane(p.page[j]), bad);
            // the half's tokens: places in_page ..; at the sequence's end the last one again
            const int room = last - min(tok + 16 * j, last & ~15); // >= 0
            const uint16_t *at = base + (int64_t(page) * page_step + int64_t(p.in_page[j]) * token_step);
            if constexpr (!V) key(at + int64_t(min(c, room)) * token_step, j);
            else {
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    load_words<F::VW>(at + (int64_t(min(4 * g + n, room)) * token_step + vc), f.v[4 * j + n]);
            }
        }
    } else {
        const int mine = held_page(a.pool, p.page, bad);
        auto at = [&](int t) { // the tile's token t
            const int page = __shfl(mine, t), in = __shfl(p.in_page, t);
            return base + (int64_t(page) * page_step + int64_t(in) * token_step);
        };
        if constexpr (!V) {
#pragma unroll
            for (int j = 0; j < 2; ++j) key(at(16 * j + c), j);
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n) load_words<F::VW>(at(4 * g + (n & 3) + 16 * (n >> 2)) + vc, f.v[n]);
        }
    }
}

// V of channel jj of the lane for its 8 tokens, as a product's operand.
template <int DP>
__device__ __forceinline__ u32x4a few_v(const FewTile<DP> &f, int jj) {
    u32x4a x;
    const uint32_t sel = jj & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int n = 0; n < 4; ++n) x[n] = __builtin_amdgcn_perm(f.v[2 * n + 1][jj >> 1], f.v[2 * n][jj >> 1], sel);
    return x;
}

template <int DP, bool HALF, int NC, bool HALVES, bool CAUSAL>
__global__ __launch_bounds__(kPagedThreads) __attribute__((amdgpu_waves_per_eu(Few<DP>::template Occ<NC, CAUSAL>, Few<DP>::template Occ<NC, CAUSAL>))) void
paged_few_kernel(PagedAttnArgs a) {
    using F = Few<DP>;
    __shared__ float joint[kPagedWaves][16][F::Row];
    const int lane = lane_id(), c = lane & 15, g = lane >> 4, wave = int(threadIdx.x) >> 6;
    int split, head, tile, seq;
    find_work(a, split, head, tile, seq);
    Rows r;
    find_rows(a, seq, split, tile, 16 * NC, r);
    const int r0 = 16 * NC * tile;
    if (r0 >= r.count || !r.used) return;
    const int low = row_limit(a, r, r0); // the tile's fewest tokens
    const int32_t *table = a.batch.table + (a.shared ? 0 : int64_t(seq) * a.batch.table_stride);
    const uint16_t *kh = a.pool.k + int64_t(head) * a.pool.k_head;
    const uint16_t *vh = a.pool.v + int64_t(head) * a.pool.v_head;
    const int vc = min(F::C * c, a.dim - F::C);
    // the rows' queries: channels 32 i + 8 g ..; rows 16 x + c
    u32x4a q[NC][F::KS];
    int limit[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
        const int row = r0 + 16 * x + c, rr = min(row, r.count - 1);
        limit[x] = row_limit(a, r, row);
        const uint16_t *qr = a.q.p + int64_t(row_token(a, r, rr)) * a.q.token +
                             int64_t(head * a.group + rr % a.group) * a.q.head;
#pragma unroll
        for (int i = 0; i < F::KS; ++i) {
            const int ch = 32 * i + 8 * g;
            q[x][i] = row < r.count && ch < a.dim ? *reinterpret_cast<const u32x4a *>(qr + ch) : u32x4a{0, 0, 0, 0};
        }
    }
    f32x4 acc[NC][F::C];
    float m[NC], l[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
        m[x] = -__builtin_inff();
        l[x] = 0.0f;
#pragma unroll
        for (int j = 0; j < F::C; ++j) acc[x][j] = f32x4{0, 0, 0, 0};
    }
    bool bad = false;
    constexpr int Step = 32 * kPagedWaves;
    const int last = r.t1 - 1;

    // one tile; once K has given its scores, `keys_done` may request others in its place
    // (CUT: some row does not see some of these tokens)
    auto work = [&](auto cut_tile, FewTile<DP> &f, int tok, auto keys_done) {
        constexpr bool cut = decltype(cut_tile)::value;
        if (a.dim != DP) { // channels past head_dim: zero, as their queries are
#pragma unroll
            for (int i = 0; i < F::KS; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (32 * i + 8 * g >= a.dim) f.k[j][i] = u32x4a{0, 0, 0, 0};
        }
        bool wild = false;
        const bool now = cut && tok + 32 > min(low, r.t1);
        if (now) {
            if constexpr (CAUSAL) {
                bool w = false;
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int k = 0; k < F::VW; ++k) w |= wild2<HALF>(f.v[n][k]);
                wild = __ballot(w) != 0;
            } else { // the rows see the same tokens: the others' values are zero
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    if (tok + 4 * g + (n & 3) + 16 * (n >> 2) >= r.t1)
#pragma unroll
                        for (int k = 0; k < F::VW; ++k) f.v[n][k] = 0;
            }
        }
        f32x4 s[NC][2];
#pragma unroll
        for (int x = 0; x < NC; ++x) {
            s[x][0] = s[x][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < F::KS; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) s[x][j] = mfma16<HALF>(f.k[j][i], q[x][i], s[x][j]);
        }
        keys_done();
        u32x4a hi[NC], lo[NC];
#pragma unroll
        for (int x = 0; x < NC; ++x) {
            float p[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) p[n] = s[x][n >> 2][n & 3] * a.scale2;
            if (now) {
                const int seen = min(limit[x], r.t1) - (tok + 4 * g); // lane's token n is seen if off(n) < seen
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    if ((n & 3) + 16 * (n >> 2) >= seen) p[n] = -__builtin_inff();
            }
            float t = p[0];
#pragma unroll
            for (int n = 1; n < 8; ++n) t = fmaxf(t, p[n]);
            t = fmaxf(t, __shfl_xor(t, 16));
            t = fmaxf(t, __shfl_xor(t, 32));
            const float mn = fmaxf(m[x], t);
            const float base = mn == -__builtin_inff() ? 0.0f : mn;
            const float alpha = exp2_f32(m[x] - base);
            m[x] = mn;
            l[x] *= alpha;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                p[n] = exp2_f32(p[n] - base);
                l[x] += p[n];
            }
#pragma unroll
            for (int j = 0; j < F::C; ++j) acc[x][j] *= alpha;
            // P as the sum of two 16-bit numbers (16 bits of it, so that an
            // output's error stays its own rounding; the pass waits for memory)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                hi[x][n] = pack2<HALF>(p[2 * n], p[2 * n + 1]);
                lo[x][n] = pack2<HALF>(p[2 * n] - low_f32<HALF>(hi[x][n]), p[2 * n + 1] - high_f32<HALF>(hi[x][n]));
            }
        }
        using W = Wild<HALF>;
#pragma unroll
        for (int j = 0; j < F::C; ++j) {
            u32x4a v = few_v<DP>(f, j);
            if constexpr (CAUSAL && cut) {
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n] = W::without(v[n]);
            }
#pragma unroll
            for (int x = 0; x < NC; ++x) {
                acc[x][j] = mfma16<HALF>(v, hi[x], acc[x][j]);
                acc[x][j] = mfma16<HALF>(v, lo[x], acc[x][j]);
            }
        }
        if constexpr (CAUSAL && cut) {
            if (!wild) return;
#pragma unroll
            for (int j = 0; j < F::C; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    u32x4a v = few_v<DP>(f, j), sees;
#pragma unroll
                    for (int n = 0; n < 4; ++n) v[n] = W::only(v[n], s != 0);
#pragma unroll
                    for (int x = 0; x < NC; ++x) {
                        const int seen = min(limit[x], r.t1) - (tok + 4 * g);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const int at = ((2 * n) & 3) + 16 * (n >> 1);
                            sees[n] = (at < seen ? W::One : 0u) | (at + 1 < seen ? W::One << 16 : 0u);
                        }
                        f32x4 z = {0, 0, 0, 0};
                        z = mfma16<HALF>(v, sees, z);
#pragma unroll
                        for (int i = 0; i < 4; ++i) z[i] = W::reach(z[i], s != 0);
                        acc[x][j] += z;
                        __builtin_amdgcn_sched_barrier(0); // (one at a time: registers)
                    }
                }
        }
    };

    int tok = r.t0 + 32 * wave;
    if (tok < r.t1) {
        // the places of the tile after the one that is requested are on their way
        FewPlaces<HALVES> next;
        FewTile<DP> f0;
        auto keys = [&](int t, FewTile<DP> &f) { few_load<DP, HALVES, false>(a, kh, t, last, vc, next, bad, f); };
        auto values = [&](int t, FewTile<DP> &f) { few_load<DP, HALVES, true>(a, vh, t, last, vc, next, bad, f); };
        auto places = [&](int t) { few_places<HALVES>(a.pool, table, t, last, next); };
        places(tok);
        keys(tok, f0);
        values(tok, f0);
        places(tok + Step);
        using Whole = std::integral_constant<bool, false>;
        using Cut = std::integral_constant<bool, true>;
        const int whole = min(low, r.t1) - 32; // tiles up to here are seen whole by every row
        if constexpr (F::template Ahead<NC>) {
            FewTile<DP> f1;
            auto next_tile = [&](FewTile<DP> &f) {
                keys(tok + Step, f);
                values(tok + Step, f);
                places(tok + 2 * Step);
            };
            auto turn = [&](FewTile<DP> &f, FewTile<DP> &g) {
                next_tile(g);
                if (CAUSAL && tok <= whole) work(Whole{}, f, tok, [] {});
                else work(Cut{}, f, tok, [] {});
                tok += Step;
                return tok < r.t1;
            };
            while (turn(f0, f1) && turn(f1, f0)) {}
        } else {
            auto turn = [&](auto cut) {
                work(cut, f0, tok, [&] {
                    if constexpr (F::Early) keys(tok + Step, f0);
                });
                tok += Step;
                if (tok >= r.t1) return false;
                if constexpr (!F::Early) keys(tok, f0);
                values(tok, f0);
                places(tok + Step);
                return true;
            };
            bool more = true;
            if constexpr (CAUSAL)
                while (more && tok <= whole) more = turn(Whole{});
            while (more) more = turn(Cut{});
        }
        if (bad) atomicOr(a.status, kStPage);
    }
    // the waves' states to LDS, 16 rows at a time: lane (c, g) holds row c,
    // channels min(C (4 g + i), dim - C) + j
#pragma unroll
    for (int x = 0; x < NC; ++x) {
        const int rows = min(16, r.count - r0 - 16 * x);
        if (rows <= 0) return;
        l[x] += __shfl_xor(l[x], 16);
        l[x] += __shfl_xor(l[x], 32);
        for (int d0 = 0; d0 < a.dim; d0 += F::JC) {
            if (x > 0 || d0 > 0) __syncthreads();
            if (g == 0 && d0 == 0) {
                joint[wave][c][F::JC] = m[x];
                joint[wave][c][F::JC + 1] = l[x];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ch = min(F::C * (4 * g + i), a.dim - F::C) - d0;
#pragma unroll
                for (int j = 0; j < F::C; ++j)
                    if (F::JC == DP || uint32_t(ch + j) < uint32_t(F::JC)) joint[wave][c][ch + j] = acc[x][j][i];
            }
            __syncthreads();
            const int nd = min(F::JC, a.dim - d0);
            for (int i = int(threadIdx.x); i < rows * nd; i += kPagedThreads) {
                const int rr = i / nd, d = i - rr * nd;
                float M = -__builtin_inff();
#pragma unroll
                for (int w = 0; w < kPagedWaves; ++w) M = fmaxf(M, joint[w][rr][F::JC]);
                const float base = M == -__builtin_inff() ? 0.0f : M;
                float L = 0.0f, A = 0.0f;
#pragma unroll
                for (int w = 0; w < kPagedWaves; ++w) {
                    const float e = exp2_f32(joint[w][rr][F::JC] - base);
                    // a wave without tokens for the row (l 0) adds nothing
                    const float lw = joint[w][rr][F::JC + 1];
                    L += lw == 0.0f ? 0.0f : lw * e;
                    A += lw == 0.0f ? 0.0f : joint[w][rr][d] * e;
                }
                write_state<HALF>(a, r, head, split, r0 + 16 * x + rr, d0 + d, M, L, A);
            }
        }
    }
}

// threadIdx.x as the compiler does not know it: what follows from it is computed
// where it is used instead of being held in registers across a loop.
__device__ __forceinline__ int thread_here() {
    int t = int(threadIdx.x);
    asm volatile("" : "+v"(t));
    return t;
}

// -------------------------------------------------------------- many rows --
// 128 or 256 query rows per workgroup, 32 per wave (32 x 32 x 16 products):
// prompts in chunks, draft tokens, and the rows of a whole batch against a
// shared prefix. A tile of tokens (64 up to head_dim 128, 32 above) is staged
// in LDS, once for all rows: pages as they are, containers decoded on the way
// (SRC 1). Rows of K are read from LDS as they lie; V's operand, four tokens of
// one channel per lane, by the transposing read. P is rounded once to 16 bits:
// the second product would else cost twice, and the error that this leaves in
// an output (a sum of independent roundings) is as large as the output's own
// rounding.
//
// Bound: the vector ALU (per tile and wave 32 exponentials at a quarter of its
// rate, their arguments, maxima and sums) and the matrix cores, in turn. The
// tile after next is on its way in registers and the next one in another part
// of LDS while a tile is worked on; a workgroup's waves meet once per tile
// (containers in two parts: twice, the escapes being written over their
// elements between). Four waves of two workgroups share a CU, or eight of one,
// two per SIMD, so that one's products run beside the other's exponentials.
// Measured: chunks of two prompts (of up to 2,048 tokens, up to 16,384 seen, 32
// heads of 128 channels) 0.9 PFLOP/s in 573 us, the matrix cores busy 45 % of it
// and the vector ALU 51 %;
// four waves per workgroup 665, a maximum per 32 tokens 860. 256 rows over
// 65,536 compressed tokens of 8 heads of 128 channels: 138 us (matrix cores 23
// %, vector ALU 37 %; with the decode's two barriers per tile 140 to 143, with
// two tiles on their way, which spills at 128 channels, 175).
template <int DP, int NW>
struct Many {
    static constexpr int T = 64 * NW;                         // threads
    static constexpr int Rows = 32 * NW;                      // query rows
    static constexpr int KT = tile_tokens(DP);
    static constexpr int ST = KT / 32;                        // score tiles
    static constexpr int KS = DP / 16;                        // steps of 16 channels
    static constexpr int CT = DP / 32;                        // channel tiles of the output
    static constexpr int KR = DP + 8;                         // LDS elements per row of K: rows 4 banks apart
    static constexpr int VR = DP + (DP % 64 == 0 ? 32 : 0);   // of V: four rows 16 banks apart
    static constexpr int PR = DP / 8;                         // 16-byte pieces per row
    static constexpr int Occ = DP <= 128 ? 2 : 1;             // waves per SIMD that the registers allow
    static constexpr int Pieces = KT * PR;
    static constexpr int NP = (Pieces + T - 1) / T;           // pieces per thread (pages)
    // containers: a thread keeps to one column of 8 channels, RP rows a pass
    static constexpr int RP = T / PR < KT ? T / PR : KT;
    static constexpr int NR = (KT + RP - 1) / RP;
};

template <int DP>
struct alignas(16) ManyBuf {
    uint16_t k[Many<DP, 4>::KT * Many<DP, 4>::KR];
    uint16_t v[Many<DP, 4>::KT * Many<DP, 4>::VR];
};
// Pages: two halves, and where K and V of the tokens of tiles on their way
// begin (bytes). Containers: three parts where the LDS of the workgroups of a
// CU allows it, else two.
template <int DP, int SRC, int NW>
struct alignas(16) ManyLds {
    static constexpr int Bufs = SRC == 1 && (NW == 8 || DP <= 64 || DP > 128) ? 3 : 2;
    ManyBuf<DP> buf[Bufs];
    longlong2 row[2][SRC == 0 ? Many<DP, 4>::KT : 1];
};

typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t any_u32 __attribute__((aligned(1)));

// A load from global memory at any alignment. (A pointer that comes from lanes
// says nothing of where it points; a flat load would count as an LDS access too,
// and the barriers would wait for it.)
template <class T>
__device__ __forceinline__ T global_at(const void *p) {
    return *(const __attribute__((address_space(1))) T *)(uintptr_t)(p);
}

// An octet of channels of a coded tensor is kept in LDS as the decoder of the
// decode kernels gives it: dword p holds channels p and p + 4. The queries are
// put in the same order, and the outputs back from it.
__device__ __forceinline__ int octet_place(int ch) { return (ch & ~7) | ((ch & 3) << 1) | ((ch >> 2) & 1); }

// 8 channels of one row of a run, as they lie in the container.
struct CodedOctet {
    uint2 sm; // sign/mantissa bytes (a plain block: the first 8 bytes)
    uint2 c;  // x: the codes, at its upper end (a plain block: the other 8 bytes)
};

// A run, read through the scalar cache (the same in every lane; the tables do
// not change while a prefix lives).
typedef const __attribute__((address_space(4))) PrefixSeg c_seg;
__device__ __forceinline__ PrefixSeg seg_at(const PrefixSeg *segs, int i) {
    c_seg *p = (c_seg *)(uintptr_t)(segs + i);
    PrefixSeg s;
    s.data = p->data;
    s.esc = p->esc;
    s.n_esc = p->n_esc;
    s.mode = p->mode;
    s.n_tokens = p->n_tokens;
    s.row0 = p->row0;
    s.rows = p->rows;
    s.dst = p->dst;
    s.more = p->more;
    s.n_more = p->n_more;
    return s;
}

// The same from a run's dwords, one per lane.
constexpr int SegWords = int(sizeof(PrefixSeg) / 4);
__device__ __forceinline__ PrefixSeg seg_of(uint32_t w) {
    uint32_t d[SegWords];
#pragma unroll
    for (int i = 0; i < SegWords; ++i) d[i] = uint32_t(__builtin_amdgcn_readlane(int(w), i));
    return __builtin_bit_cast(PrefixSeg, d);
}

// The octet from channel ch of row `row` of a run; `plain`: its mode is 0. The
// codes come as the dword that ends with them (bytes of the block before them
// in front), so that no load reaches past the block.
__device__ __forceinline__ void load_octet(const PrefixSeg &s, bool plain, int dim, int row, int ch, CodedOctet &o) {
    const uint32_t e = uint32_t((s.row0 + row) * dim + ch); // element of the block
    if (plain) {
        const any_u32x2 a = global_at<any_u32x2>(s.data + 2 * e),
                        b = global_at<any_u32x2>(s.data + (2 * e + 8));
        o.sm = make_uint2(a.x, a.y);
        o.c = make_uint2(b.x, b.y);
        return;
    }
    const any_u32x2 sm = global_at<any_u32x2>(s.data + (uint32_t(dim) + e));
    o.sm = make_uint2(sm.x, sm.y);
    const uint8_t *codes = s.data + (dim + s.n_tokens * dim + s.mode - 4);
    o.c = make_uint2(global_at<any_u32>(codes + (e >> 3) * uint32_t(s.mode)), 0);
}

// The octet's BF16 words in octet order (escapes come after), from its base
// words (channels p and p + 4 of the block's base exponents, shifted by 7).
template <int MODE>
__device__ __forceinline__ u32x4a decode_octet(const CodedOctet &o, const uint32_t (&bp)[4], uint32_t smm) {
    uint32_t cw, t[4];
    if constexpr (MODE == 4) cw = o.c.x;
    else if constexpr (MODE == 2) cw = __builtin_amdgcn_perm(o.c.x, o.c.x, 0x0c030c02u);
    else cw = ((o.c.x >> 8) & 0xFFFu) | ((o.c.x >> 4) & 0x0FFF0000u);
    team::octet_exponents<MODE>(cw, bp, t);
    return u32x4a{team::team_pair(o.sm.x, o.sm.y, 0, t[0], smm), team::team_pair(o.sm.x, o.sm.y, 1, t[1], smm),
                  team::team_pair(o.sm.x, o.sm.y, 2, t[2], smm), team::team_pair(o.sm.x, o.sm.y, 3, t[3], smm)};
}
__device__ __forceinline__ u32x4a plain_octet(const CodedOctet &o) {
    const uint4 x = team::raw_octet(make_uint4(o.sm.x, o.sm.y, o.c.x, o.c.y));
    return u32x4a{x.x, x.y, x.z, x.w};
}
__device__ __forceinline__ void base_words(uint2 base, uint32_t (&bp)[4]) {
#pragma unroll
    for (uint32_t p = 0; p < 4; ++p)
        bp[p] = __builtin_amdgcn_perm(base.y, base.x, 0x0c000c00u | ((4u + p) << 16) | p) << 7;
}

// A tile of a container tensor on its way: the rows of its first run in
// registers (pass k: row RP k + the thread's row), and its first escape
// records, one per thread.
template <int DP, int NW>
struct CodedTile {
    CodedOctet o[Many<DP, NW>::NR];
    uint2 base;
    uint32_t rec;
};

// The thread's column and row of a pass; rows per pass.
struct Column {
    int ch, row, step;
};

// Whether a run fills the tile and its rows the passes (the usual case): then a
// pass is a fixed step of the streams after the one before.
template <int DP, int NW>
__device__ __forceinline__ bool whole_run(const PrefixSeg &s, int dim) {
    using S = Many<DP, NW>;
    return s.rows == S::KT && dim == DP && S::T % S::PR == 0 && S::T <= S::Pieces;
}

template <int DP, int NW>
__device__ __forceinline__ void coded_load(const PrefixSeg &s, int dim, const Column &at, CodedTile<DP, NW> &t) {
    using S = Many<DP, NW>;
    const int tid = thread_here();
    t.rec = global_at<uint32_t>(s.esc + max(min(tid, s.n_esc - 1), 0));
    // (a plain block has no base exponents; it starts with at least a row)
    const any_u32x2 b = global_at<any_u32x2>(s.data + uint32_t(at.ch));
    t.base = make_uint2(b.x, b.y);
    if (s.mode != 0 && whole_run<DP, NW>(s, dim)) {
        const uint32_t e0 = uint32_t(8 * tid); // element of the run
        const uint8_t *sm = s.data + (DP + s.row0 * DP),
                      *codes = s.data + (DP + s.n_tokens * DP + s.row0 * (DP / 8) * s.mode + s.mode - 4);
        const uint32_t c0 = uint32_t(tid) * uint32_t(s.mode);
#pragma unroll
        for (int k = 0; k < S::NR; ++k) {
            const any_u32x2 x = global_at<any_u32x2>(sm + 8 * S::T * k + e0);
            t.o[k].sm = make_uint2(x.x, x.y);
            t.o[k].c = make_uint2(global_at<any_u32>(codes + S::T * k * s.mode + c0), 0);
        }
        return;
    }
    const int lastp = s.rows - 1;
    if (s.mode != 0) {
#pragma unroll
        for (int k = 0; k < S::NR; ++k) load_octet(s, false, dim, min(at.row + at.step * k, lastp), at.ch, t.o[k]);
    } else {
#pragma unroll
        for (int k = 0; k < S::NR; ++k) load_octet(s, true, dim, min(at.row + at.step * k, lastp), at.ch, t.o[k]);
    }
}

// The run's rows to LDS rows of R elements; V: the tile's other rows are zero
// (a run of the tile's end: the prefix's end) before further runs are written.
template <int DP, int NW, int R, bool V>
__device__ __forceinline__ void coded_store(const PrefixSeg &s, const PrefixSeg *segs, int dim, const Column &at,
                                            const CodedTile<DP, NW> &t, uint16_t *lds) {
    using S = Many<DP, NW>;
    const uint32_t smm = wave::sm_mask_vgpr();
    const bool mine = at.row < at.step; // (threads past the whole rows of a pass have none)
    auto put = [&](auto octet) {
        if (whole_run<DP, NW>(s, dim)) {
            uint16_t *to = lds + at.row * R + at.ch;
#pragma unroll
            for (int k = 0; k < S::NR; ++k) *reinterpret_cast<u32x4a *>(to + k * S::RP * R) = octet(k);
            return;
        }
#pragma unroll
        for (int k = 0; k < S::NR; ++k) {
            const int row = at.row + at.step * k;
            const u32x4a w = octet(k);
            if (mine && row < s.rows) *reinterpret_cast<u32x4a *>(lds + row * R + at.ch) = w;
            else if (V && mine && row < S::KT && s.n_more == 0)
                *reinterpret_cast<u32x4a *>(lds + row * R + at.ch) = u32x4a{0, 0, 0, 0};
        }
    };
    uint32_t bp[4];
    base_words(t.base, bp);
    if (s.mode == 4) put([&](int k) { return decode_octet<4>(t.o[k], bp, smm); });
    else if (s.mode == 2) put([&](int k) { return decode_octet<2>(t.o[k], bp, smm); });
    else if (s.mode == 3) put([&](int k) { return decode_octet<3>(t.o[k], bp, smm); });
    else put([&](int k) { return plain_octet(t.o[k]); });
    if (s.n_more == 0) return;
    // blocks that end inside the tile: their rows are read here
    int end = s.rows;
    for (int i = 0; i < s.n_more; ++i) {
        const PrefixSeg g = seg_at(segs, s.more + i);
        end = g.dst + g.rows;
        uint2 base = make_uint2(0, 0);
        if (g.mode != 0) {
            const any_u32x2 b = global_at<any_u32x2>(g.data + at.ch);
            base = make_uint2(b.x, b.y);
        }
        base_words(base, bp);
        for (int row = at.row; mine && row < g.rows; row += at.step) {
            CodedOctet o;
            load_octet(g, g.mode == 0, dim, row, at.ch, o);
            *reinterpret_cast<u32x4a *>(lds + (g.dst + row) * R + at.ch) =
                g.mode == 4   ? decode_octet<4>(o, bp, smm)
                : g.mode == 2 ? decode_octet<2>(o, bp, smm)
                : g.mode == 3 ? decode_octet<3>(o, bp, smm)
                              : plain_octet(o);
        }
    }
    if (V)
        for (int row = end + at.row; mine && row < S::KT; row += at.step)
            *reinterpret_cast<u32x4a *>(lds + row * R + at.ch) = u32x4a{0, 0, 0, 0};
}

// An escape record of a run over its element.
template <int R>
__device__ __forceinline__ void patch_one(const PrefixSeg &s, int dim, uint32_t rec, uint16_t *lds) {
    const int e = int(rec & 0xFFFFu), row = e / dim - s.row0;
    if (uint32_t(row) < uint32_t(s.rows)) // (a damaged container's records)
        lds[(s.dst + row) * R + octet_place(e - (row + s.row0) * dim)] = uint16_t(rec >> 16);
}
template <int DP, int NW, int R>
__device__ __forceinline__ void coded_patch(const PrefixSeg &s, const PrefixSeg *segs, int dim,
                                            const CodedTile<DP, NW> &t,
                                            uint16_t *lds) {
    const int tid = int(threadIdx.x);
    if (tid < s.n_esc) patch_one<R>(s, dim, t.rec, lds);
    for (int i = tid + 64 * NW; i < s.n_esc; i += 64 * NW) patch_one<R>(s, dim, global_at<uint32_t>(s.esc + i), lds);
    for (int k = 0; k < s.n_more; ++k) {
        const PrefixSeg g = seg_at(segs, s.more + k);
        for (int i = tid; i < g.n_esc; i += 64 * NW) patch_one<R>(g, dim, global_at<uint32_t>(g.esc + i), lds);
    }
}

template <int DP, bool HALF, int SRC, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(Many<DP, NW>::Occ, Many<DP, NW>::Occ))) void
paged_many_kernel(PagedAttnArgs a) {
    using S = Many<DP, NW>;
    extern __shared__ __align__(16) uint8_t many_lds[];
    using Lds = ManyLds<DP, SRC, NW>;
    Lds &lds = *reinterpret_cast<Lds *>(many_lds);
    const int tid = int(threadIdx.x), lane = lane_id(), wave = tid >> 6, c = lane & 31, h = lane >> 5;
    int split, head, tile, seq;
    find_work(a, split, head, tile, seq);
    Rows r;
    find_rows(a, seq, split, tile, S::Rows, r);
    if (S::Rows * tile >= r.count || !r.used) return;
    const int r0 = 32 * (NW * tile + wave);
    const int row = r0 + c, limit = row_limit(a, r, row);
    const bool busy = r0 < r.count;
    const int low = row_limit(a, r, min(r0, r.count - 1)); // the wave's fewest tokens
    const int wg_low = row_limit(a, r, S::Rows * tile);
    const int32_t *table = a.batch.table + (a.shared ? 0 : int64_t(seq) * a.batch.table_stride);
    const uint16_t *kh = a.pool.k + int64_t(head) * a.pool.k_head;
    const uint16_t *vh = a.pool.v + int64_t(head) * a.pool.v_head;
    // channels past head_dim: K's are zero (they meet zero queries), V's feed outputs that nobody reads
    for (int i = tid; i < Lds::Bufs * S::KT * (DP - a.dim); i += S::T) {
        const int t = i / (DP - a.dim), d = a.dim + i - t * (DP - a.dim), b = t / S::KT;
        lds.buf[b].k[(t - b * S::KT) * S::KR + d] = 0;
        lds.buf[b].v[(t - b * S::KT) * S::VR + d] = 0;
    }
    // the queries, their sign turned where the scale is negative
    const float scale2 = fabsf(a.scale2);
    u32x4a q[S::KS];
    {
        const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;
        const int rr = min(row, r.count - 1);
        const uint16_t *qr = a.q.p + int64_t(row_token(a, r, rr)) * a.q.token +
                             int64_t(head * a.group + rr % a.group) * a.q.head;
#pragma unroll
        for (int i = 0; i < S::KS; ++i) q[i] = *reinterpret_cast<const u32x4a *>(qr + min(16 * i + 8 * h, a.dim - 8));
#pragma unroll
        for (int i = 0; i < S::KS; ++i) {
            if constexpr (SRC == 1) {
                const uint4 x = team::raw_octet(make_uint4(q[i][0], q[i][1], q[i][2], q[i][3]));
                q[i] = u32x4a{x.x, x.y, x.z, x.w};
            }
            const bool none = row >= r.count || 16 * i + 8 * h >= a.dim;
#pragma unroll
            for (int n = 0; n < 4; ++n) q[i][n] = none ? 0u : q[i][n] ^ flip;
        }
    }
    f32x16 acc[S::CT];
#pragma unroll
    for (int j = 0; j < S::CT; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    // ---- one tile, from its half of LDS (CUT: some row of the workgroup does
    // not see all of it). All its scores first: one maximum, one branch, and
    // the second half's exponentials run beside the first half's products.
    auto work = [&](auto cut, int tok, const ManyBuf<DP> &buf, bool wild) {
        constexpr bool CUT = decltype(cut)::value;
        f32x16 s[S::ST];
#pragma unroll
        for (int t = 0; t < S::ST; ++t) {
            s[t] = f32x16{};
#pragma unroll
            for (int i = 0; i < S::KS; ++i) {
                const u32x4a kf = *reinterpret_cast<const u32x4a *>(buf.k + (32 * t + c) * S::KR + 16 * i + 8 * h);
                s[t] = mfma32<HALF>(kf, q[i], s[t]);
            }
        }
        // a few rows of K ahead of the products (else each product waits for its own)
        constexpr int Reads = S::KS * S::ST, Deep = Reads < 6 ? Reads : 6;
        __builtin_amdgcn_sched_group_barrier(0x100, Deep, 0);
#pragma unroll
        for (int i = 0; i < Reads - Deep; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, Deep, 0);
        // element i of s[t]: token tok + 32 t + 8 (i / 4) + 4 h + i % 4
        if (CUT && tok + S::KT > min(low, r.t1)) {
            const int seen = min(limit, r.t1) - tok - 4 * h;
#pragma unroll
            for (int t = 0; t < S::ST; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * t + 8 * (i >> 2) + (i & 3) >= seen) s[t][i] = -__builtin_inff();
        }
        float mt = s[0][0];
#pragma unroll
        for (int t = 0; t < S::ST; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[t][i]);
        mt = fmaxf(mt, __shfl_xor(mt, 32)) * scale2;
        // m follows the maximum only when that is 2^8 above it: until then the
        // weights are at most 2^8 (and as exact), and the sums keep their scale
        if (__ballot(mt > m + 8.0f) != 0) {
            const float mn = fmaxf(m, mt);
            const float alpha = exp2_f32(m - (mn == -__builtin_inff() ? 0.0f : mn));
            l *= alpha;
#pragma unroll
            for (int j = 0; j < S::CT; ++j) acc[j] *= alpha;
            m = mn;
        }
        const float base = m == -__builtin_inff() ? 0.0f : m;
        // V: lane group lane / 16 reads channels 16 (group % 2) .. of tokens 4 (group / 2) ..
        const uint16_t *vl = buf.v + ((lane & 15) >> 2) * S::VR + 4 * h * S::VR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        auto value = [&](int k, int j) { // the operand of tokens 16 k .. and channels 32 j ..
            const uint16_t *at = vl + 16 * k * S::VR + 32 * j;
            const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at));
            const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + 8 * S::VR));
            const uint2 x = __builtin_bit_cast(uint2, v0), y = __builtin_bit_cast(uint2, v1);
            return u32x4a{x.x, x.y, y.x, y.y};
        };
        using W = Wild<HALF>;
        float sum[2] = {0.0f, 0.0f};
        __builtin_amdgcn_s_setprio(1); // (the other wave of the SIMD is at its scores: chunks of prompts 608 -> 597 us)
#pragma unroll
        for (int k = 0; k < 2 * S::ST; ++k) { // 16 tokens
            f32x16 &sk = s[k >> 1];
            u32x4a p;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = 8 * (k & 1) + 2 * n;
                const float p0 = exp2_f32(__builtin_fmaf(sk[i], scale2, -base)),
                            p1 = exp2_f32(__builtin_fmaf(sk[i + 1], scale2, -base));
                sum[0] += p0;
                sum[1] += p1;
                p[n] = pack2<HALF>(p0, p1);
            }
#pragma unroll
            for (int j = 0; j < S::CT; ++j) {
                u32x4a v = value(k, j);
                if constexpr (CUT && SRC == 0) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) v[n] = W::without(v[n]);
                }
                acc[j] = mfma32<HALF>(v, p, acc[j]);
            }
        }
        l += sum[0] + sum[1];
        __builtin_amdgcn_s_setprio(0);
        if constexpr (CUT && SRC == 0) {
            if (!wild) return;
            const int seen = min(limit, r.t1) - tok - 4 * h;
#pragma unroll
            for (int j = 0; j < S::CT; ++j)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    f32x16 z = {};
#pragma unroll
                    for (int k = 0; k < 2 * S::ST; ++k) {
                        u32x4a v = value(k, j), sees;
#pragma unroll
                        for (int n = 0; n < 4; ++n) { // tokens at and at + 1 of the tile (plus 4 h)
                            const int at = 16 * k + 8 * (n >> 1) + ((2 * n) & 3);
                            sees[n] = (at < seen ? W::One : 0u) | (at + 1 < seen ? W::One << 16 : 0u);
                            v[n] = W::only(v[n], g != 0);
                        }
                        z = mfma32<HALF>(v, sees, z);
                        __builtin_amdgcn_sched_barrier(0); // (one at a time: registers)
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = W::reach(z[i], g != 0);
                    acc[j] += z;
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };
    using Whole = std::integral_constant<bool, false>;
    using Cut = std::integral_constant<bool, true>;

    if (r.t0 < r.t1) {
        if constexpr (SRC == 0) {
            u32x4a kn[S::NP], vn[S::NP]; // the rows of a tile on their way
            bool bad = false;
            int2 place; // of one token of the tile after it
            auto find = [&](int tok) {
                const int t = min(tok + min(tid, S::KT - 1), r.t1 - 1);
                const int col = page_of(a.pool, t);
                place.x = table[col];
                place.y = t - col * a.pool.page_tokens;
            };
            auto publish = [&](int slot) {
                if (tid >= S::KT) return;
                const int64_t page = held_page(a.pool, place.x, bad);
                lds.row[slot][tid] = make_longlong2(2 * (page * a.pool.k_page + int64_t(place.y) * a.pool.k_token),
                                                    2 * (page * a.pool.v_page + int64_t(place.y) * a.pool.v_token));
            };
            auto request = [&](int slot) {
                const int here = thread_here();
                const char *kc = nullptr, *vc = nullptr;
#pragma unroll
                for (int k = 0; k < S::NP; ++k) {
                    const int o = min(here + S::T * k, S::Pieces - 1), t = o / S::PR;
                    if (k == 0 || S::T % S::PR != 0) { // (else the same channels every time)
                        const int ch = min(8 * (o - t * S::PR), a.dim - 8);
                        kc = reinterpret_cast<const char *>(kh + ch);
                        vc = reinterpret_cast<const char *>(vh + ch);
                    }
                    const longlong2 at = lds.row[slot][t];
                    kn[k] = *reinterpret_cast<const u32x4a *>(kc + at.x);
                    vn[k] = *reinterpret_cast<const u32x4a *>(vc + at.y);
                }
            };
            // Tokens past the split's end: V is zero. Returns whether the tile
            // holds an infinity or NaN in V where rows see different tokens of it.
            auto store = [&](ManyBuf<DP> &buf, int tok) {
                bool w = false;
                if (tok + S::KT > wg_low || tok + S::KT > r.t1) {
#pragma unroll
                    for (int k = 0; k < S::NP; ++k) {
                        const int t = (tid + S::T * k) / S::PR;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            vn[k][i] = tok + t < r.t1 ? vn[k][i] : 0u;
                            w |= wild2<HALF>(vn[k][i]);
                        }
                    }
                    w &= tok + S::KT > wg_low;
                }
                const int here = thread_here();
                auto put = [&](int k) {
                    const int o = here + S::T * k, t = o / S::PR, ch = 8 * (o - t * S::PR);
                    if (S::Pieces % S::T != 0 && o >= S::Pieces) return;
                    *reinterpret_cast<u32x4a *>(buf.k + t * S::KR + ch) = kn[k];
                    *reinterpret_cast<u32x4a *>(buf.v + t * S::VR + ch) = vn[k];
                };
                if (a.dim == DP) {
#pragma unroll
                    for (int k = 0; k < S::NP; ++k) put(k);
                } else {
#pragma unroll
                    for (int k = 0; k < S::NP; ++k)
                        if (8 * ((here + S::T * k) % S::PR) < a.dim) put(k);
                }
                return w;
            };
            int tok = r.t0, b = 0;
            find(tok);
            publish(0);
            find(tok + S::KT);
            publish(1);
            find(tok + 2 * S::KT);
            __syncthreads();
            request(0);
            bool w = store(lds.buf[0], tok);
            request(1);
            bool wild = __syncthreads_or(w) != 0;
            // works on the tile at tok and makes the next one ready; false at the end
            auto turn = [&](auto cut) {
                if (busy) work(cut, tok, lds.buf[b], wild);
                if (tok + S::KT >= r.t1) return false;
                w = store(lds.buf[b ^ 1], tok + S::KT);
                publish(b); // the tile after next; its rows are requested after the barrier
                find(tok + 3 * S::KT);
                if (tok + 2 * S::KT > wg_low) wild = __syncthreads_or(w) != 0;
                else team::team_sync(); // (the loads on their way stay on their way)
                tok += S::KT;
                if (tok + S::KT < r.t1) request(b);
                b ^= 1;
                return true;
            };
            // tiles that every row sees whole, then the others
            bool more = true;
            while (more && tok + S::KT <= min(wg_low, r.t1)) more = turn(Whole{});
            while (more) more = turn(Cut{});
            if (bad) atomicOr(a.status, kStPage);
        } else {
            const PrefixSeg *ks = a.px[2 * head].segs, *vs = a.px[2 * head + 1].segs;
            const int pr = a.dim / 8, last = (r.len - 1) / S::KT;
            const Column at{8 * (tid % pr), tid / pr, min(S::T / pr, S::KT)};
            CodedTile<DP, NW> kt, vt;
            // the tile's first runs, and the next tile's on their way, a dword
            // per lane (through the scalar cache they would hold up the LDS
            // reads of the tile being worked on, which wait on the same count)
            PrefixSeg k0, v0;
            uint32_t k1, v1;
            auto fetch = [&](int t) {
                k1 = reinterpret_cast<const uint32_t *>(ks + min(t, last))[min(lane, SegWords - 1)];
                v1 = reinterpret_cast<const uint32_t *>(vs + min(t, last))[min(lane, SegWords - 1)];
            };
            auto request = [&](int t) {
                k0 = seg_of(k1);
                v0 = seg_of(v1);
                coded_load<DP, NW>(k0, a.dim, at, kt);
                coded_load<DP, NW>(v0, a.dim, at, vt);
                fetch(t + 1);
            };
            int t = r.t0 / S::KT;
            fetch(t);
            request(t);
            auto put = [&](ManyBuf<DP> &buf) {
                coded_store<DP, NW, S::KR, false>(k0, ks, a.dim, at, kt, buf.k);
                coded_store<DP, NW, S::VR, true>(v0, vs, a.dim, at, vt, buf.v);
            };
            auto patch = [&](ManyBuf<DP> &buf, bool more) { // and the next tile's rows requested
                coded_patch<DP, NW, S::KR>(k0, ks, a.dim, kt, buf.k);
                coded_patch<DP, NW, S::VR>(v0, vs, a.dim, vt, buf.v);
                if (more) request(++t);
            };
            // (team_sync: loads on their way stay on their way)
            if constexpr (Lds::Bufs == 3) {
                // The part that the next tile is put in was last read two tiles
                // ago, and its escapes are written before the barrier that the
                // tile's own work waits for: one barrier per tile.
                put(lds.buf[0]);
                team::team_sync();
                patch(lds.buf[0], r.t0 + S::KT < r.t1);
                for (int tok = r.t0, b = 0; tok < r.t1; tok += S::KT) {
                    const int next = b == 2 ? 0 : b + 1;
                    const bool more = tok + S::KT < r.t1;
                    if (more) put(lds.buf[next]);
                    team::team_sync();
                    if (more) patch(lds.buf[next], tok + 2 * S::KT < r.t1);
                    if (busy) work(Cut{}, tok, lds.buf[b], false);
                    b = next;
                }
            } else {
                for (int tok = r.t0, b = 0; tok < r.t1; tok += S::KT, b ^= 1) {
                    put(lds.buf[b]);
                    team::team_sync();
                    patch(lds.buf[b], tok + S::KT < r.t1);
                    team::team_sync();
                    if (busy) work(Cut{}, tok, lds.buf[b], false);
                }
            }
        }
    }
    if (!busy) return;
    l += __shfl_xor(l, 32);
    if (row >= r.count) return;
    // lane (c, h): row c, places 32 j + 8 i + 4 h .. + 3 of the channels
    const int64_t slot = state_slot(a, r, head, split, row);
    const int64_t tok = row_token(a, r, row);
    const int hq = head * a.group + row % a.group;
    if (h == 0) {
        if (a.direct) {
            if (a.lse != nullptr) a.lse[tok * (a.n_kv * a.group) + hq] = log_sum(m, l);
        } else {
            a.ml[2 * slot] = m;
            a.ml[2 * slot + 1] = l;
        }
    }
#pragma unroll
    for (int j = 0; j < S::CT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ch = 32 * j + 8 * i + 4 * h;
            if (ch >= a.dim) continue;
            const float x0 = acc[j][4 * i], x1 = acc[j][4 * i + 1], x2 = acc[j][4 * i + 2], x3 = acc[j][4 * i + 3];
            if constexpr (SRC == 1) { // octet order: channels 2 h, 2 h + 4, 2 h + 1, 2 h + 5 (never direct)
                float *o = a.acc + slot * a.dim + (32 * j + 8 * i + 2 * h);
                *reinterpret_cast<float2 *>(o) = make_float2(x0, x2);
                *reinterpret_cast<float2 *>(o + 4) = make_float2(x1, x3);
            } else if (a.direct) {
                uint2 w;
                w.x = pack2<HALF>(finish(x0, l), finish(x1, l));
                w.y = pack2<HALF>(finish(x2, l), finish(x3, l));
                *reinterpret_cast<uint2 *>(a.out.p + tok * a.out.token + int64_t(hq) * a.out.head + ch) = w;
            } else {
                *reinterpret_cast<float4 *>(a.acc + slot * a.dim + ch) = make_float4(x0, x1, x2, x3);
            }
        }
}

} // namespace paged
} // namespace kvexp_dev
