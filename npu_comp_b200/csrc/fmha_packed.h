// Internal interface of the packed / paged attention kernel (fmha_packed.cu),
// shared with the decode path (paged_decode.cu).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace npub {

// K and V of a call: packed rows (table == nullptr) or pages.
struct KvSource {
    const void *k, *v;
    int64_t ldk, ldv;        // rows: element strides
    const int32_t* table;    // pages: [batch, max_pages] page ids, row stride ldt
    int64_t ldt;
    int max_pages, n_pages, page_size;
    int common;              // pages, paged_decode: the first `common` keys of all sequences are looked up in row 0
};

struct PackedArgs {
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    KvSource kv;
    const int32_t* cu;    // [batch + 1]; null: one row per sequence
    const int32_t* lens;  // pages: keys of each sequence (shared-prefix phase: of each row)
    int total_q, batch, heads, kv_heads, head_dim;
    int shared;           // > 0: shared-prefix phase, the first `shared` keys of row 0's pages for all rows
    float scale;
    int causal;
    // splits > 1 (or shared): fp32 partials instead of out
    int tiles;            // row tiles of an item: 1, 2, or 0 (chosen by the number of items)
    int dual;             // partials, tiles == 1: an item's keys in two halves, two partials for each split
    int splits;           // equal ranges of every sequence's keys from `first` on
    int first, split0;    // split0: index of split 0 among the partials
    float* part_o;        // [splits, total_q, heads, head_dim]
    // [splits, total_q, heads]: (row's reference score, sum of exponentials); (-inf, 0) where the row has no key
    // in the range, (-inf, 1) where all its scores there are -inf (part_o is not written then)
    float2* part_ml;
    // pages of whole numbers (null: of values): for every 16 keys, [batch, kv_heads, max_pages * page_size / 16],
    // (log2(e) scale s_k, log2 s_v), with which a score's sum of products becomes the exponent of its weight times s_v;
    // (NaN, 0) where a scale is not finite;
    // part_ml's references are such exponents
    const float2* key_scale;
};

int fmha_packed(const PackedArgs& a, cudaStream_t st);
// Items (per kv head) of `tiles` row tiles: at most this many for rows in ascending offsets; max_new > 0: for sequences
// of no more rows (estimates only).
int64_t fmha_packed_items(int total_q, int batch, int heads, int kv_heads, int max_new, int tiles);
// 4-D map of a page pool [n_pages, kv_heads, page_size, head_dim], box {64, box_rows, 1, 1}, 128-byte swizzle.
int make_tmap_pages(CUtensorMap* m, const void* base, int n_pages, int kv_heads, int page_size, int head_dim,
                    int box_rows);
// The same of 8-bit pages: whole rows, box {64 or 128, box_rows, 1, 1} with a swizzle of its width.
int make_tmap_pages_q8(CUtensorMap* m, const void* base, int n_pages, int kv_heads, int page_size, int head_dim,
                       int box_rows);

}  // namespace npub
