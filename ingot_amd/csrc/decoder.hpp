// Launch interface between the decoder-step entry points (decoder.cpp) and
// their kernels (rotary.hip, kv_pages.hip, tree_attention.hip).
#pragma once

#include "common.hpp"

namespace ingot {

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 by one multiplication: with
// 2^(s − 1) < d <= 2^s and m = ceil(2^(31 + s) / d), m·d passes 2^(31 + s) by
// less than 2^s, so n·m / 2^(31 + s) has the floor of n / d.
struct FastDiv {
    uint32_t m;
    int32_t s, d;
    FastDiv() = default;
    explicit FastDiv(int32_t v) : m(0), s(0), d(v) {
        while (((int64_t)1 << s) < v) ++s;
        m = (uint32_t)((((uint64_t)1 << (31 + s)) + (uint32_t)v - 1) / (uint32_t)v);
    }
    __device__ __forceinline__ int div(int n) const { return (int)(__umulhi((uint32_t)n << 1, m) >> s); }
};

// What a kernel reads of ingot_rocm_kv_cache (one layer), _kv_table and _kv_batch.
struct KvView {
    char *k, *v;  // of the layer
    int64_t stride_page, stride_head, stride_slot;  // elements
    const int32_t* pages;
    const int32_t* len;
    const int32_t* starts;
    const int32_t* row;  // NULL: row b is sequence b
    int32_t page_size, num_pages, kv_heads, max_pages, rows, batch, tokens;
    FastDiv by_page;

    // Row of sequence b, -1 where the table has none.
    __device__ __forceinline__ int row_of(int b) const {
        const int r = row ? row[b] : b;
        return r >= 0 && r < rows ? r : -1;
    }
    // Page of position pos of a row, -1 where there is none.
    __device__ __forceinline__ int page_of(int r, int64_t pos) const {
        if (pos < 0 || pos > 0x7FFFFFFF) return -1;
        const int p = by_page.div((int)pos);
        if (p >= max_pages) return -1;
        const int id = pages[(int64_t)r * max_pages + p];
        return id < num_pages ? id : -1;
    }
};

struct HeadsView {
    char* data;
    int64_t token, head;  // elements
};

struct RotaryView {
    const float *cos, *sin;
    const int32_t* positions;
    int64_t rows;
    int32_t half;  // rotated pairs
    int32_t interleaved, inverse;
};

hipError_t launch_rotary_table(const ingot_rocm_rotary_table_args& a, hipStream_t st);
// y = x turned; with `kv` (append) also k turned and v into the cache's slots.
struct RotaryArgs {
    RotaryView rot;
    HeadsView x, y, k, v;
    int64_t tokens;
    int32_t heads, kv_heads, dim;  // kv_heads 0: no cache
    KvView kv;
};
hipError_t launch_rotary(const RotaryArgs& a, int dtype, int cache_dtype, hipStream_t st);


// One page operation's view of the cache over all layers: a page's slots of a
// layer are `segs` runs of rows, a row being the 16-byte chunks that lie
// together for one slot (the head's, or all heads' where they are neighbours).
struct PagesView {
    char *k, *v;
    int64_t stride_layer, stride_page, stride_seg, stride_slot;  // bytes
    int32_t layers, segs, row_chunks, page_size, num_pages, rows, max_pages;
    FastDiv by_page;
    int32_t *pages, *len, *refs, *missing;
};
hipError_t launch_kv_copy(const PagesView& p, const int32_t* src, const int32_t* dst, int64_t n, hipStream_t st);
// Scratch of the two calls that hand out pages.
size_t kv_alloc_ws(int64_t n, int64_t pages);
hipError_t launch_kv_reserve(const PagesView& p, const int32_t* row, const int32_t* tokens, int n, void* ws, hipStream_t st);
hipError_t launch_kv_fork(const PagesView& p, const int32_t* src, const int32_t* dst, int n, void* ws, hipStream_t st);
hipError_t launch_kv_free(const PagesView& p, const int32_t* row, int n, hipStream_t st);
hipError_t launch_kv_compact(const PagesView& p, const int32_t* row, const int32_t* accept, const int32_t* count, int n,
                             int max_accept, int32_t* new_len, hipStream_t st);

struct TreeAttnArgs {
    KvView kv;
    HeadsView q, y;
    const uint32_t* mask;  // NULL: a chain
    int64_t mask_words;
    int32_t heads, group, dim, max_nodes, max_tokens;
    FastDiv by_group;
    int32_t q_bf16;        // q and y are bf16, else f32
    int32_t q_vec, y_vec;  // rows of q (y) allow 16-byte (4-element) accesses
    int32_t flip;          // queries are negated: scale is positive
    float scale;           // · log2(e)
    // Set by the launch: positions are cut into `splits` pieces of `chunk`, rows
    // (node, query head of the key head's group) into `row_tiles`. With `slots`
    // the device cuts them by their lengths into at most so many pieces of at
    // least `chunk`.
    int32_t chunk, splits, row_tiles, items, slots;
    int4* cuts;       // [sequence · key head][row tile] first piece, pieces, step from one to the next
    float* part_o;    // [item][row][dim] sums of a piece, not divided
    float2* part_ml;  // [item][row] running maximum (log2 units) and sum of a piece
};
// Fills the geometry and says what scratch it needs (0: one piece); then the
// pointers into it.
size_t plan_tree_attention(TreeAttnArgs& a, int cache_dtype, int num_cus);
void place_tree_attention(TreeAttnArgs& a, int cache_dtype, void* ws);
hipError_t launch_tree_attention(const TreeAttnArgs& a, int cache_dtype, hipStream_t st);

}  // namespace ingot
