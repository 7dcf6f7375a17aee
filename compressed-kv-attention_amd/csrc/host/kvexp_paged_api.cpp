// C ABI of the paged cache (include/kvexp_hip.h, "paged cache"): argument
// checks, the choice of kernel and splits, workspace layout, and the tables of
// shared prefixes kept as containers.
#include "api_common.hpp"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>

#include "../hip/paged_types.h"

using namespace kvexp_host;
using namespace kvexp_dev;

namespace kvexp_launch {
hipError_t rotate(RotateArgs a, bool half, hipStream_t s);
hipError_t paged_attention(const PagedAttnArgs &a, bool half, int tile_rows, int n_seqs, hipStream_t s);
hipError_t paged_merge(const PagedAttnArgs &a, bool half, hipStream_t s);
hipError_t prefix_segs(PrefixSeg *segs, int n, const EscJob *jobs, hipStream_t s);
} // namespace kvexp_launch

struct kvexp_hip_prefix {
    int device = 0; // (the context may be gone when the prefix goes)
    int n_heads = 0, dim = 0, seq = 0;
    DevBuf arena;
    const PrefixTensor *tensors = nullptr;
};

namespace {

constexpr int kMaxHeadDim = 256;
constexpr int64_t kThreadsMax = int64_t(UINT32_MAX);  // of a launch
constexpr int64_t kTokensMax = int64_t(1) << 30;       // of a sequence: a tile's end stays an int
constexpr int64_t kRotTokensMax = int64_t(1) << 27;    // new tokens of a rotation: its threads stay a launch's
constexpr int64_t kRotChannelsMax = int64_t(1) << 26;  // a token's channels over all heads: 16 tokens' stay an int

[[noreturn]] void bad(const std::string &msg) { fail(KVEXP_HIP_INVALID_ARGUMENT, msg); }

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

void check_dim(const char *who, int dim) {
    if (dim <= 0 || dim % 8 != 0 || dim > kMaxHeadDim)
        bad(std::string(who) + ": head_dim must be a multiple of 8 and at most 256");
}
void check_dtype(const char *who, int dtype) {
    if (dtype != KVEXP_HIP_BF16 && dtype != KVEXP_HIP_FP16) bad(std::string(who) + ": elements are BF16 or FP16");
}
void check_rows(const char *who, const char *name, const kvexp_hip_rows *r) {
    if (r == nullptr || r->data == nullptr) bad(std::string(who) + ": null " + name);
    if (!aligned(r->data, 16) || r->token % 8 != 0 || r->head % 8 != 0)
        bad(std::string(who) + ": " + name + " must be 16-byte aligned, with strides that are multiples of 8 elements");
}

RowsDev rows_in(const kvexp_hip_rows *r) { return {static_cast<const uint16_t *>(r->data), r->token, r->head}; }
RowsOut rows_out(const kvexp_hip_rows *r) {
    return {static_cast<uint16_t *>(const_cast<void *>(r->data)), r->token, r->head};
}

// t / d by multiplication for 0 <= t < 2^31: with l = ceil(log2 d),
// floor(t m / 2^(31 + l)) for m = floor(2^(31 + l) / d) + 1 (the error term
// t (m d - 2^(31 + l)) / d 2^(31 + l) stays below 1 / d). magic 0: a shift.
void division(uint32_t d, uint32_t &magic, int32_t &shift) {
    int l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    if ((d & (d - 1)) == 0) {
        magic = 0;
        shift = l;
        return;
    }
    magic = uint32_t((uint64_t(1) << (31 + l)) / d + 1);
    shift = l - 1;
}

PoolDev pool_of(const char *who, const kvexp_hip_pages *p) {
    if (p == nullptr || p->k == nullptr || p->v == nullptr) bad(std::string(who) + ": null pages");
    check_dtype(who, p->dtype);
    check_dim(who, p->dim);
    if (p->n_pages <= 0 || p->page_tokens <= 0 || p->n_heads <= 0) bad(std::string(who) + ": empty pages");
    const int64_t strides[] = {p->k_page, p->k_head, p->k_token, p->v_page, p->v_head, p->v_token};
    for (int64_t s : strides)
        if (s % 8 != 0) bad(std::string(who) + ": strides of pages must be multiples of 8 elements");
    if (!aligned(p->k, 16) || !aligned(p->v, 16)) bad(std::string(who) + ": pages must be 16-byte aligned");
    PoolDev d{};
    d.k = static_cast<uint16_t *>(p->k);
    d.v = static_cast<uint16_t *>(p->v);
    d.k_page = p->k_page, d.k_head = p->k_head, d.k_token = p->k_token;
    d.v_page = p->v_page, d.v_head = p->v_head, d.v_token = p->v_token;
    d.n_pages = p->n_pages;
    d.page_tokens = p->page_tokens;
    division(uint32_t(p->page_tokens), d.page_magic, d.page_shift);
    return d;
}

BatchDev batch_of(const char *who, const kvexp_hip_batch *b, int page_tokens, int &max_len) {
    if (b == nullptr) bad(std::string(who) + ": null batch");
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->table_width < 0) bad(std::string(who) + ": negative size");
    BatchDev d{};
    d.table = b->table;
    d.lens = b->lens;
    d.starts = b->starts;
    d.table_stride = b->table_stride;
    d.table_width = b->table_width;
    d.n_seqs = b->n_seqs;
    d.n_tokens = b->n_tokens;
    max_len = 0;
    if (b->n_tokens == 0) return d;
    if (b->n_seqs == 0) bad(std::string(who) + ": tokens of no sequence");
    if (b->lens == nullptr || (b->table == nullptr && b->table_width > 0)) bad(std::string(who) + ": null table or lens");
    if (b->n_seqs > 1 && b->table_stride < b->table_width) bad(std::string(who) + ": rows of the page table overlap");
    const int64_t most = int64_t(b->table_width) * page_tokens;
    if (most > kTokensMax) fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": a page table of more than 2^30 tokens");
    if (b->starts == nullptr) {
        if (b->n_tokens % b->n_seqs != 0)
            bad(std::string(who) + ": without starts every sequence has n_tokens / n_seqs new tokens");
        d.n_new = b->n_tokens / b->n_seqs;
        if (b->max_new > 0 && b->max_new < d.n_new) bad(std::string(who) + ": max_new below the new tokens");
        d.max_new = d.n_new;
    } else {
        d.max_new = b->max_new > 0 ? std::min(b->max_new, b->n_tokens) : b->n_tokens;
    }
    max_len = int(b->max_len > 0 ? std::min<int64_t>(b->max_len, most) : most);
    return d;
}

RopeDev rope_of(const char *who, const kvexp_hip_rope *r, const kvexp_hip_positions *p, int dim, int n_tokens) {
    RopeDev d{};
    d.n_axes = 1;
    d.scale = d.sign = 1.0f;
    if (r == nullptr) return d;
    if (r->inv_freq == nullptr || r->n_freq <= 0) bad(std::string(who) + ": a rotation without frequencies");
    if (2 * int64_t(r->n_freq) > dim) bad(std::string(who) + ": more rotated channels than head_dim");
    if (r->n_axes <= 0) bad(std::string(who) + ": a rotation without axes");
    d.freq = r->inv_freq;
    d.axes = r->axes;
    d.n_freq = r->n_freq;
    d.n_axes = r->n_axes;
    d.interleaved = r->interleaved != 0;
    d.scale = r->scale;
    if (p != nullptr) {
        d.pos = p->data;
        d.axis_stride = p->axis_stride;
        d.offset = p->offset;
        d.pos64 = p->wide != 0;
        if (p->data != nullptr && !aligned(p->data, p->wide ? 8 : 4)) bad(std::string(who) + ": unaligned positions");
        if (p->data != nullptr && r->n_axes > 1 && p->axis_stride < n_tokens)
            bad(std::string(who) + ": axes of the positions overlap");
    }
    return d;
}

void check_rotation(const char *who, int n_tokens, int64_t channels) {
    if (n_tokens > kRotTokensMax || channels > kRotChannelsMax)
        fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": more tokens or heads than a launch takes");
}

// How a call is cut.
struct Cut {
    int tile_rows = 16, row_tiles = 1, n_splits = 1, min_split = 64;
};

// Rows per (sequence, head) pick the kernel: what a workgroup of the few-row
// kernel takes (few_rows), or the many-row kernel, whose tiles go through LDS.
Cut cut_of(const kvexp_hip_ctx *ctx, int64_t rows, int64_t pairs, int max_len, int dim, bool shared, bool coded) {
    Cut c;
    if (rows > INT32_MAX / 2) fail(KVEXP_HIP_UNSUPPORTED, "paged attention: too many query rows");
    const bool many = coded || rows > few_rows(dim);
    c.tile_rows = !many ? (rows > 16 ? 32 : 16) : many_rows(dim, coded);
    // 256 rows where they are not a tenth more than tiles of 128 would have (300
    // rows, 8 x 4 over 16,000 tokens of 128 channels: 118 us in three tiles of
    // 128, 136 in two of 256; full tiles are a tenth faster with 256)
    auto padded_rows = [&](int64_t tile) { return (rows + tile - 1) / tile * tile; };
    if (c.tile_rows == 256 && 10 * padded_rows(256) > 11 * padded_rows(128)) c.tile_rows = 128;
    c.row_tiles = int((rows + c.tile_rows - 1) / c.tile_rows);
    // Few rows: splits of 512 tokens at least (one sequence of 65,536 tokens, 2
    // heads of 64 channels: 23.6 us, with 256 31.7), where that leaves eight of
    // them (one of 1,021 tokens: kernels 11.8 us with 256, 12.9 with 512); eight
    // workgroups per CU in all, of which three run at once, so that short
    // sequences' empty splits leave enough of them (64 sequences of 1K to 32K:
    // 85 us, with five 90, with sixteen 79; but four of up to 65,536 at 128
    // channels 125, 123, 136); with two products of rows six, as every split's
    // states cost twice as much (16 sequences of 8,192, 32 rows of 128 channels:
    // 77 us, with eight 83, with four 73; but 16 of up to 16,411 with up to five
    // drafts, 4 queries of 96 channels: 54, 56, 64). Many rows: 256 at least (30
    // rows over 4,096 compressed tokens: 25 us, with 512 33), and the workgroups
    // that are resident: one of 256 rows per CU, one of 128 above head_dim 128
    // (730 shared rows over 4,586 tokens of 256 channels: 73 us, for two 93), else
    // two; of unequal sequences and causal tiles twice that (12 prompts of up to
    // 3,051 tokens, 248 rows of 8 heads of 128 channels: 49 us, else 74; of 256
    // channels 120 and 192).
    c.min_split = many || max_len <= 4096 ? 256 : 512;
    const int64_t resident = c.tile_rows == 256 || dim > 128 ? 1 : 2;
    const int64_t per_cu = !many ? (c.tile_rows == 32 ? 6 : 8) : shared ? resident : 2 * resident;
    const int64_t target = int64_t(std::max(1, ctx->cu_count)) * per_cu;
    const int64_t base = std::max<int64_t>(1, pairs * c.row_tiles);
    // (many rows: no second round for a few more)
    const int64_t want = many ? std::max<int64_t>(1, target / base) : (target + base - 1) / base;
    const int64_t most = std::max<int64_t>(1, (int64_t(max_len) + c.min_split - 1) / c.min_split);
    c.n_splits = int(std::max<int64_t>(1, std::min<int64_t>({want, most, 256})));
    // the splits of the longest sequence the call may hold: shorter ones take fewer
    const int64_t even = (int64_t(max_len) + c.n_splits - 1) / c.n_splits;
    c.min_split = int(std::max<int64_t>(c.min_split, (even + 63) / 64 * 64));
    return c;
}

// Threads of the launch over `pairs` (sequence, head) pairs.
int64_t threads_of(const Cut &c, int64_t pairs) {
    if (pairs > kThreadsMax) return INT64_MAX;
    const int64_t per = int64_t(c.row_tiles) * c.n_splits; // < 2^31 * 2^8
    const int64_t threads = c.tile_rows == 256 ? 512 : 256;
    return per > kThreadsMax / threads / std::max<int64_t>(1, pairs) ? INT64_MAX : per * pairs * threads;
}

struct Call {
    PagedAttnArgs own{}, shared{};
    Cut cut, shared_cut;
    bool has_shared = false, half = false;
    int64_t slots = 0, shared_slots = 0;
    size_t at_ml = 0, at_shared_acc = 0, at_shared_ml = 0, bytes = 0;
};

size_t padded(size_t n) { return (n + 255u) & ~size_t(255); }

Call plan_call(kvexp_hip_ctx *ctx, const kvexp_hip_pages *pages, const kvexp_hip_batch *batch,
               const kvexp_hip_shared *shared, int n_q_heads) {
    const char *who = "kvexp_hip_paged_attention";
    Call c;
    PagedAttnArgs &a = c.own;
    a.pool = pool_of(who, pages);
    int max_len;
    a.batch = batch_of(who, batch, pages->page_tokens, max_len);
    if (n_q_heads <= 0 || n_q_heads % pages->n_heads != 0)
        bad(std::string(who) + ": query heads must be a multiple of the cache's heads");
    c.half = pages->dtype == KVEXP_HIP_FP16;
    a.n_kv = pages->n_heads;
    a.group = n_q_heads / pages->n_heads;
    a.dim = pages->dim;
    c.has_shared = shared != nullptr;
    if (c.has_shared) {
        const bool xkv = shared->xkv != nullptr;
        if (xkv == (shared->table != nullptr)) bad(std::string(who) + ": a shared prefix is containers or pages");
        if (xkv) {
            const kvexp_hip_prefix &p = *shared->xkv;
            if (c.half) bad(std::string(who) + ": containers hold BF16, the pages FP16");
            if (p.n_heads != a.n_kv || p.dim != a.dim) bad(std::string(who) + ": the prefix has other heads or head_dim");
            if (shared->n_tokens != p.seq) bad(std::string(who) + ": n_tokens must be the prefix's");
        } else {
            if (shared->n_tokens <= 0) bad(std::string(who) + ": an empty shared prefix");
            if (shared->n_tokens > kTokensMax)
                fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": a shared prefix of more than 2^30 tokens");
            if (int64_t(shared->table_width) * pages->page_tokens < shared->n_tokens)
                bad(std::string(who) + ": the shared prefix's table is shorter than its tokens");
        }
    }
    if (a.batch.n_tokens == 0) return c;
    if (ctx == nullptr) bad(std::string(who) + ": null context");
    if (c.has_shared && shared->xkv != nullptr && shared->xkv->device != ctx->device)
        bad(std::string(who) + ": the prefix is on another device");
    const int64_t rows = int64_t(a.batch.max_new) * a.group;
    c.cut = cut_of(ctx, rows, int64_t(a.batch.n_seqs) * a.n_kv, max_len, a.dim, false, false);
    // (the merge: a wave per query row)
    if (threads_of(c.cut, int64_t(a.batch.n_seqs) * a.n_kv) > kThreadsMax ||
        int64_t(a.batch.n_tokens) * n_q_heads > kThreadsMax / 64 - 4)
        fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": more sequences or query rows than a launch takes");
    a.row_tiles = c.cut.row_tiles;
    a.n_splits = c.cut.n_splits;
    a.min_split = c.cut.min_split;
    a.max_rows = a.batch.n_tokens * a.group;
    a.direct = !c.has_shared && a.n_splits == 1;
    if (!a.direct) {
        c.slots = int64_t(a.n_kv) * a.n_splits * a.max_rows;
        c.at_ml = padded(size_t(c.slots) * size_t(a.dim) * sizeof(float));
        c.bytes = c.at_ml + padded(size_t(c.slots) * 2 * sizeof(float));
    }
    if (c.has_shared) {
        PagedAttnArgs &p = c.shared;
        p = a;
        p.shared = 1;
        p.direct = 0;
        p.len = shared->n_tokens;
        const bool xkv = shared->xkv != nullptr;
        c.shared_cut = cut_of(ctx, int64_t(a.batch.n_tokens) * a.group, a.n_kv, p.len, a.dim, true, xkv);
        if (threads_of(c.shared_cut, a.n_kv) > kThreadsMax)
            fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": more query rows than a launch takes");
        p.row_tiles = c.shared_cut.row_tiles;
        p.n_splits = c.shared_cut.n_splits;
        p.min_split = c.shared_cut.min_split;
        if (xkv) p.px = shared->xkv->tensors;
        else {
            p.batch.table = shared->table;
            p.batch.table_width = shared->table_width;
        }
        c.shared_slots = int64_t(p.n_kv) * p.n_splits * p.max_rows;
        c.at_shared_acc = c.bytes;
        c.at_shared_ml = c.at_shared_acc + padded(size_t(c.shared_slots) * size_t(a.dim) * sizeof(float));
        c.bytes = c.at_shared_ml + padded(size_t(c.shared_slots) * 2 * sizeof(float));
        a.s_splits = p.n_splits;
        a.s_rows = p.max_rows;
        a.s_min_split = p.min_split;
        a.s_len = p.len;
    }
    return c;
}

// The tables of a prefix kept as containers: reads the block indexes (checked
// block by block), cuts every tensor's tokens into the kernel's tiles and
// those at block ends, and fills in addresses and escape records on the GPU.
void build_prefix(kvexp_hip_ctx *ctx, kvexp_hip_prefix &p, const kvexp_hip_head *heads, hipStream_t s) {
    const int n = 2 * p.n_heads, kt = tile_tokens(p.dim), tiles = (p.seq + kt - 1) / kt;
    std::vector<EscJob> jobs;
    std::vector<size_t> at; // a tensor's first entry in the index arrays
    size_t total = 0;
    for (int i = 0; i < n; ++i) {
        const kvexp_hip_head &h = heads[i / 2];
        EscJob j{};
        j.blob = i & 1 ? h.v_xkv : h.k_xkv;
        j.bytes = i & 1 ? h.v_bytes : h.k_bytes;
        j.offs = i & 1 ? h.v_offsets : h.k_offsets;
        j.first = i & 1 ? h.v_first_token : h.k_first_token;
        j.n_blocks = i & 1 ? h.v_n_blocks : h.k_n_blocks;
        j.dim = p.dim;
        at.push_back(total);
        total += size_t(j.n_blocks) + 1;
        jobs.push_back(j);
    }
    if (total > size_t(INT32_MAX)) fail(KVEXP_HIP_UNSUPPORTED, "kvexp_hip_prefix_create: too many blocks");
    std::vector<int32_t> e0(total), first(total);
    struct SyncOnExit { // buffers and host arrays outlive the work queued on them
        hipStream_t s;
        ~SyncOnExit() { (void)hipStreamSynchronize(s); }
    };
    const size_t jobs_b = jobs.size() * sizeof(EscJob);
    {
        DevBuf buf(&ctx->pool, jobs_b + (1 + 2 * total) * sizeof(int32_t));
        auto *words = reinterpret_cast<int32_t *>(buf.as<uint8_t>() + jobs_b);
        std::vector<uint8_t> up(jobs_b + sizeof(uint32_t), 0);
        SyncOnExit sync{s};
        for (int i = 0; i < n; ++i) {
            EscJob j = jobs[size_t(i)];
            j.esc0 = words + 1 + at[size_t(i)];
            j.first_out = words + 1 + total + at[size_t(i)];
            std::memcpy(up.data() + size_t(i) * sizeof j, &j, sizeof j);
        }
        HIPX(hipMemcpyAsync(buf.p, up.data(), up.size(), hipMemcpyHostToDevice, s));
        HIPX(kvexp_launch::esc_start(buf.as<EscJob>(), n, reinterpret_cast<uint32_t *>(words), s));
        // (and what the tables below take at most: a tile's or a block's start begins a run)
        const size_t runs = size_t(n) * size_t(tiles) + total;
        auto *host = static_cast<int32_t *>(pinned_staging(
            ctx, std::max((1 + 2 * total) * sizeof(int32_t),
                          size_t(n) * (sizeof(PrefixTensor) + sizeof(EscJob)) +
                              total * (sizeof(int2) + sizeof(int32_t)) + runs * sizeof(PrefixSeg) + 8 * padded(1))));
        HIPX(hipMemcpyAsync(host, words, (1 + 2 * total) * sizeof(int32_t), hipMemcpyDeviceToHost, s));
        HIPX(hipStreamSynchronize(s));
        if (host[0] != 0) fail(KVEXP_HIP_FORMAT_ERROR, status_message(uint32_t(host[0])));
        std::copy(host + 1, host + 1 + total, e0.begin());
        std::copy(host + 1 + total, host + 1 + 2 * total, first.begin());
    }
    // the runs of every tensor: each tile's first one, then the further ones
    std::vector<PrefixSeg> segs, more;
    std::vector<size_t> seg_at, pos_at;
    std::vector<int2> blocks;
    size_t pos_total = 0;
    for (int i = 0; i < n; ++i) {
        const int nb = jobs[size_t(i)].n_blocks;
        const int32_t *f = first.data() + at[size_t(i)];
        for (int b = 0; b < nb; ++b)
            if (f[b] < 0 || f[b + 1] <= f[b] || f[0] != 0)
                fail(KVEXP_HIP_FORMAT_ERROR, "xkv block index does not match the container");
        if (f[nb] < p.seq) fail(KVEXP_HIP_FORMAT_ERROR, "xkv ran out of tokens");
        seg_at.push_back(segs.size());
        more.clear();
        int b = 0, tok = 0;
        for (int t = 0; t < tiles; ++t) {
            const int end = std::min(p.seq, (t + 1) * kt);
            const size_t head = segs.size();
            for (bool is_first = true; tok < end; is_first = false) {
                while (f[b + 1] <= tok) ++b;
                PrefixSeg g{};
                g.n_esc = i; // (see prefix_segs_kernel)
                g.mode = b;
                g.row0 = tok - f[b];
                g.rows = std::min(end, int(f[b + 1])) - tok;
                g.dst = tok - t * kt;
                tok += g.rows;
                if (is_first) {
                    g.more = int32_t(size_t(tiles) + more.size());
                    segs.push_back(g);
                } else {
                    more.push_back(g);
                    ++segs[head].n_more;
                }
            }
        }
        segs.insert(segs.end(), more.begin(), more.end());
        for (b = 0; b < nb; ++b) blocks.push_back(make_int2(i, b));
        pos_at.push_back(pos_total);
        pos_total += size_t(e0[at[size_t(i)] + size_t(nb)]);
    }
    if (segs.size() > size_t(INT32_MAX) || blocks.size() > size_t(INT32_MAX))
        fail(KVEXP_HIP_UNSUPPORTED, "kvexp_hip_prefix_create: too many blocks");
    // one allocation: what the host uploads, then the escape records
    const size_t o_tensors = padded(sizeof(uint32_t)), o_jobs = o_tensors + padded(size_t(n) * sizeof(PrefixTensor)),
                 o_blocks = o_jobs + padded(jobs_b), o_e0 = o_blocks + padded(blocks.size() * sizeof(int2)),
                 o_segs = o_e0 + padded(total * sizeof(int32_t)),
                 o_pos = o_segs + padded(segs.size() * sizeof(PrefixSeg));
    // (and one more: a run without records reads the one where its own would be)
    const size_t pos_b = (pos_total + 1) * sizeof(uint32_t);
    p.arena = DevBuf(o_pos + pos_b);
    uint8_t *d = p.arena.as<uint8_t>();
    // (in pinned memory, whose last use above is over: a copy from other memory
    // took 340 us at 16 tensors of 65,536 tokens, this one 20)
    auto *image = static_cast<uint8_t *>(pinned_staging(ctx, o_pos));
    std::memset(image, 0, o_tensors); // the status word
    std::vector<PrefixTensor> tensors(static_cast<size_t>(n));
    for (int i = 0; i < n; ++i) {
        EscJob &j = jobs[size_t(i)];
        j.esc0 = reinterpret_cast<int32_t *>(d + o_e0) + at[size_t(i)];
        j.pos = reinterpret_cast<uint32_t *>(d + o_pos) + pos_at[size_t(i)];
        tensors[size_t(i)].segs = reinterpret_cast<const PrefixSeg *>(d + o_segs) + seg_at[size_t(i)];
    }
    std::memcpy(image + o_tensors, tensors.data(), tensors.size() * sizeof(PrefixTensor));
    std::memcpy(image + o_jobs, jobs.data(), jobs_b);
    std::memcpy(image + o_blocks, blocks.data(), blocks.size() * sizeof(int2));
    std::memcpy(image + o_e0, e0.data(), total * sizeof(int32_t));
    std::memcpy(image + o_segs, segs.data(), segs.size() * sizeof(PrefixSeg));
    SyncOnExit sync{s};
    HIPX(hipMemcpyAsync(d, image, o_pos, hipMemcpyHostToDevice, s));
    HIPX(hipMemsetAsync(d + o_pos, 0, pos_b, s));
    auto *st = reinterpret_cast<uint32_t *>(d);
    const auto *dj = reinterpret_cast<const EscJob *>(d + o_jobs);
    HIPX(kvexp_launch::esc_pos(dj, reinterpret_cast<const int2 *>(d + o_blocks), int(blocks.size()), st, s));
    HIPX(kvexp_launch::prefix_segs(reinterpret_cast<PrefixSeg *>(d + o_segs), int(segs.size()), dj, s));
    check_status_word(ctx, st, s);
    p.tensors = reinterpret_cast<const PrefixTensor *>(d + o_tensors);
}

} // namespace

extern "C" {

int kvexp_hip_rope_rows(kvexp_hip_ctx *ctx, const kvexp_hip_rope *rope, const kvexp_hip_positions *positions,
                        const kvexp_hip_rows *x, const kvexp_hip_rows *out, int n_tokens, int n_heads, int dim,
                        int dtype, int inverse, void *stream) {
    return guarded([&] {
        const char *who = "kvexp_hip_rope_rows";
        if (rope == nullptr) bad(std::string(who) + ": a rotation without frequencies");
        check_dtype(who, dtype);
        check_dim(who, dim);
        if (n_tokens < 0 || n_heads <= 0) bad(std::string(who) + ": empty rows");
        RotateArgs a{};
        a.rope = rope_of(who, rope, positions, dim, n_tokens);
        check_rotation(who, n_tokens, int64_t(n_heads) * dim);
        if (n_tokens == 0) return;
        check_rows(who, "x", x);
        check_rows(who, "out", out);
        a.rope.sign = inverse ? -1.0f : 1.0f;
        a.q = rows_in(x);
        a.q_out = rows_out(out);
        a.n_q = n_heads;
        a.n_tokens = n_tokens;
        a.dim = dim;
        if (ctx == nullptr) bad(std::string(who) + ": null context");
        DeviceGuard g(ctx->device);
        HIPX(kvexp_launch::rotate(a, dtype == KVEXP_HIP_FP16, static_cast<hipStream_t>(stream)));
    });
}

int kvexp_hip_paged_append(kvexp_hip_ctx *ctx, const kvexp_hip_pages *pages, const kvexp_hip_batch *batch,
                           const kvexp_hip_rows *k, const kvexp_hip_rows *v, const kvexp_hip_rope *rope,
                           const kvexp_hip_positions *positions, const kvexp_hip_rows *q, const kvexp_hip_rows *q_out,
                           int n_q_heads, uint32_t *d_status, void *stream) {
    return guarded([&] {
        const char *who = "kvexp_hip_paged_append";
        RotateArgs a{};
        a.pool = pool_of(who, pages);
        int max_len;
        a.batch = batch_of(who, batch, pages->page_tokens, max_len);
        a.rope = rope_of(who, rope, positions, pages->dim, a.batch.n_tokens);
        if ((q == nullptr) != (q_out == nullptr)) bad(std::string(who) + ": q and q_out go together");
        if (q != nullptr && rope == nullptr) bad(std::string(who) + ": queries without a rotation");
        if (q != nullptr && n_q_heads <= 0) bad(std::string(who) + ": no query heads");
        check_rotation(who, a.batch.n_tokens, (int64_t(q != nullptr ? n_q_heads : 0) + 2 * int64_t(pages->n_heads)) * pages->dim);
        if (d_status == nullptr) bad(std::string(who) + ": null status word");
        if (a.batch.n_tokens == 0) return;
        check_rows(who, "k", k);
        check_rows(who, "v", v);
        a.k = rows_in(k);
        a.v = rows_in(v);
        a.n_kv = pages->n_heads;
        if (q != nullptr) {
            check_rows(who, "q", q);
            check_rows(who, "q_out", q_out);
            a.q = rows_in(q);
            a.q_out = rows_out(q_out);
            a.n_q = n_q_heads;
        }
        a.n_tokens = a.batch.n_tokens;
        a.dim = pages->dim;
        a.status = d_status;
        if (ctx == nullptr) bad(std::string(who) + ": null context");
        DeviceGuard g(ctx->device);
        HIPX(kvexp_launch::rotate(a, pages->dtype == KVEXP_HIP_FP16, static_cast<hipStream_t>(stream)));
    });
}

int kvexp_hip_prefix_create(kvexp_hip_ctx *ctx, const kvexp_hip_head *heads, int n_heads, int dim, void *stream,
                            kvexp_hip_prefix **out) {
    return guarded([&] {
        const char *who = "kvexp_hip_prefix_create";
        if (out == nullptr) bad(std::string(who) + ": null output");
        *out = nullptr;
        if (heads == nullptr || n_heads <= 0) bad(std::string(who) + ": bad argument");
        check_dim(who, dim);
        const int seq = heads[0].seq;
        if (seq <= 0) bad(std::string(who) + ": an empty shared prefix");
        if (seq > kTokensMax) fail(KVEXP_HIP_UNSUPPORTED, std::string(who) + ": a shared prefix of more than 2^30 tokens");
        for (int h = 0; h < n_heads; ++h) {
            const kvexp_hip_head &H = heads[h];
            if (H.k_xkv == nullptr || H.v_xkv == nullptr || H.k_offsets == nullptr || H.v_offsets == nullptr ||
                H.k_first_token == nullptr || H.v_first_token == nullptr || H.k_n_blocks <= 0 || H.v_n_blocks <= 0)
                bad(std::string(who) + ": a head without containers and their block indexes");
            if (H.seq != seq) bad(std::string(who) + ": heads of different lengths");
        }
        if (ctx == nullptr) bad(std::string(who) + ": null context");
        DeviceGuard g(ctx->device);
        auto *p = new kvexp_hip_prefix();
        try {
            p->device = ctx->device;
            p->n_heads = n_heads;
            p->dim = dim;
            p->seq = seq;
            build_prefix(ctx, *p, heads, static_cast<hipStream_t>(stream));
        } catch (...) {
            delete p;
            throw;
        }
        *out = p;
    });
}

int kvexp_hip_prefix_destroy(kvexp_hip_prefix *prefix) {
    return guarded([&] {
        if (prefix == nullptr) return;
        DeviceGuard g(prefix->device);
        delete prefix;
    });
}

int64_t kvexp_hip_paged_attention_workspace(kvexp_hip_ctx *ctx, const kvexp_hip_pages *pages,
                                            const kvexp_hip_batch *batch, const kvexp_hip_shared *shared,
                                            int n_q_heads) {
    int64_t n = -1;
    (void)guarded([&] { n = int64_t(plan_call(ctx, pages, batch, shared, n_q_heads).bytes); });
    return n;
}

int kvexp_hip_paged_attention(kvexp_hip_ctx *ctx, const kvexp_hip_pages *pages, const kvexp_hip_batch *batch,
                              const kvexp_hip_shared *shared, const kvexp_hip_rows *q, int n_q_heads, float scale,
                              const kvexp_hip_rows *out, float *d_lse, void *workspace, size_t workspace_bytes,
                              uint32_t *d_status, void *stream) {
    return guarded([&] {
        const char *who = "kvexp_hip_paged_attention";
        // never 0, which times a masked place's -inf is no number: the least
        // normal number instead (with products q . k up to 2^100 the weights
        // are those of scale 0 to 2^-26)
        float scale2 = float(double(scale) * 1.4426950408889634074);
        if (!std::isfinite(scale2)) bad(std::string(who) + ": the scale is not finite, or past float's range");
        if (std::fabs(scale2) < FLT_MIN) scale2 = std::copysign(FLT_MIN, scale2);
        if (d_status == nullptr) bad(std::string(who) + ": null status word");
        if (batch != nullptr && batch->n_tokens > 0) {
            check_rows(who, "q", q);
            check_rows(who, "out", out);
        }
        Call c = plan_call(ctx, pages, batch, shared, n_q_heads);
        if (c.own.batch.n_tokens == 0) return;
        if (c.bytes > 0 && (workspace == nullptr || !aligned(workspace, 16)))
            bad(std::string(who) + ": the workspace must be 16-byte aligned");
        if (workspace_bytes < c.bytes)
            fail(KVEXP_HIP_CAPACITY, std::string(who) + ": workspace below kvexp_hip_paged_attention_workspace");
        auto *w = static_cast<uint8_t *>(workspace);
        PagedAttnArgs &a = c.own;
        a.q = rows_in(q);
        a.out = rows_out(out);
        a.lse = d_lse;
        a.scale2 = scale2;
        a.status = d_status;
        a.acc = reinterpret_cast<float *>(w);
        a.ml = reinterpret_cast<float *>(w + c.at_ml);
        DeviceGuard g(ctx->device);
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (c.has_shared) {
            PagedAttnArgs &p = c.shared;
            p.q = a.q;
            p.scale2 = scale2;
            p.status = d_status;
            p.acc = reinterpret_cast<float *>(w + c.at_shared_acc);
            p.ml = reinterpret_cast<float *>(w + c.at_shared_ml);
            a.s_acc = p.acc;
            a.s_ml = p.ml;
            HIPX(kvexp_launch::paged_attention(p, c.half, c.shared_cut.tile_rows, 1, s));
        }
        HIPX(kvexp_launch::paged_attention(a, c.half, c.cut.tile_rows, a.batch.n_seqs, s));
        if (!a.direct) HIPX(kvexp_launch::paged_merge(a, c.half, s));
    });
}

int kvexp_hip_paged_status(kvexp_hip_ctx *ctx, uint32_t *d_status, void *stream) {
    return guarded([&] {
        if (ctx == nullptr || d_status == nullptr) bad("kvexp_hip_paged_status: null argument");
        DeviceGuard g(ctx->device);
        hipStream_t s = static_cast<hipStream_t>(stream);
        const uint32_t st = read_result(ctx, nullptr, d_status, nullptr, s);
        if (st == 0u) return;
        HIPX(hipMemsetAsync(d_status, 0, sizeof(uint32_t), s));
        HIPX(hipStreamSynchronize(s));
        if (st & kStPage) fail(KVEXP_HIP_FORMAT_ERROR, "a page table names a page outside the pool");
        if (st & kStLength)
            fail(KVEXP_HIP_FORMAT_ERROR, "a length past its page table, or more new tokens than max_new");
        fail(KVEXP_HIP_FORMAT_ERROR, "paged cache error");
    });
}

} // extern "C"
