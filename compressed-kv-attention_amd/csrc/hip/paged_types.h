// Descriptors of the paged-cache operators, shared by the host entries and the
// gfx950 kernels.
#pragma once

#include <stdint.h>

namespace kvexp_dev {

// Status bits the paged kernels raise in the caller's status word.
enum : uint32_t {
    kStPage = 1u << 8,   // a page number outside the pool
    kStLength = 1u << 9, // a length past the page table, or new tokens past max_new
};

// A pool of pages: page p, head h, token t of the page at
// p * page + h * head + t * token elements, channels contiguous.
struct PoolDev {
    uint16_t *k, *v;
    int64_t k_page, k_head, k_token;
    int64_t v_page, v_head, v_token;
    int32_t n_pages, page_tokens;
    uint32_t page_magic; // page_tokens as a multiplier (page_of); 0 for a page of one token
    int32_t page_shift;
};

// A batch of sequences over the pool. New tokens of sequence b: rows
// [starts[b], starts[b + 1]) of the call's tensors, or n_new rows each where
// starts is null.
struct BatchDev {
    const int32_t *table; // [n_seqs, table_width] pages
    const int32_t *lens;  // tokens of each sequence, the new ones included
    const int32_t *starts;
    int64_t table_stride;
    int32_t table_width, n_seqs, n_tokens, n_new, max_new;
    int32_t pad;
};

// Rows [token, head] of dim channels.
struct RowsDev {
    const uint16_t *p;
    int64_t token, head;
};
struct RowsOut {
    uint16_t *p;
    int64_t token, head;
};

struct RopeDev {
    const float *freq;   // [n_freq]
    const uint8_t *axes; // [n_freq] axis of each frequency, or null: axis 0
    const void *pos;     // [n_axes, n_tokens], int32 or int64; null: a token's place plus offset
    int64_t axis_stride; // elements
    int64_t offset;
    int32_t pos64;
    int32_t n_freq, n_axes;
    int32_t interleaved;
    float scale;
    float sign; // -1: the rotation back
};

// One call of the rotation kernel: up to three sets of heads per token, the
// first two rotated, the last copied.
struct RotateArgs {
    RowsDev q, k, v;
    RowsOut q_out;
    int32_t n_q, n_kv; // heads; n_kv 0: no append
    int32_t n_tokens, dim;
    int32_t tokens_per_group;
    int32_t pad;
    RopeDev rope;
    PoolDev pool;
    BatchDev batch;
    uint32_t *status;
};

// A run of rows of one block of a container that lie in one tile of the
// shared prefix (tile_tokens).
struct PrefixSeg {
    const uint8_t *data; // the block past its header
    const uint32_t *esc; // escape records of these rows
    int32_t n_esc;
    int32_t mode;        // 0, 2, 3, 4
    int32_t n_tokens;    // of the block
    int32_t row0;        // first row, in the block
    int32_t rows;
    int32_t dst;         // first row in the tile
    int32_t more, n_more; // further runs of the tile (blocks that end inside it): first and count
};

// One tensor (K or V of one head) of a shared prefix kept as containers: the
// first run of every tile, then the further ones.
struct PrefixTensor {
    const PrefixSeg *segs;
};

// The attention calls. Partial states: slot (row, split) holds m, l (in the
// base-2 exponent's units) and dim sums; `acc` row-major [slot][dim], `ml`
// [slot][2]; slots [head][split][token row, query head of the group].
struct PagedAttnArgs {
    PoolDev pool;
    BatchDev batch;
    RowsDev q;
    RowsOut out;
    float *lse;       // [n_tokens, n_heads] or null
    int32_t n_kv, group, dim;
    float scale2;     // scale * log2(e)
    int32_t n_splits; // slots per row
    int32_t min_split;
    int32_t direct;   // one split: the kernel writes out itself
    int32_t row_tiles;
    int32_t shared;   // rows of all sequences against one table of `len` tokens
    int32_t len;
    int32_t max_rows; // query rows of a KV head in the call: slot stride
    float *acc, *ml;
    uint32_t *status;
    const PrefixTensor *px; // [2 n_kv] (K, V of each head), shared prefixes kept as containers
    // the merge: slots of the shared part (0: none)
    const float *s_acc, *s_ml;
    int32_t s_splits, s_rows, s_min_split, s_len;
};

// Tokens of a tile of the many-row kernel.
constexpr int tile_tokens(int dim) { return dim <= 128 ? 64 : 32; }
// Query rows of a workgroup of the few-row kernel, at most: 16, or 32 in two
// products where the registers hold them.
constexpr int few_rows(int dim) { return dim <= 128 ? 32 : 16; }
// Of the many-row kernel, at most: 128, or 256 where eight waves' registers
// hold the outputs (and, for containers, the coded rows on their way).
constexpr int many_rows(int dim, bool coded) { return dim <= (coded ? 128 : 192) ? 256 : 128; }
template <int DP>
constexpr int kFewRowsAt = few_rows(DP);

} // namespace kvexp_dev
