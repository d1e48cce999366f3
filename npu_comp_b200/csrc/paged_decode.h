// Internal interface of the few-row paged attention and the combination of
// partial results (paged_decode.cu).
#pragma once

#include "fmha_packed.h"

namespace npub {

constexpr int kPagedDecodeRows = 16;  // rows per kv head that paged_decode takes

constexpr int kPagedDecodeCluster = 8;  // ranges that a cluster combines

// a.splits equal ranges of every sequence's keys from a.first on: partials a.split0 + s when a.part_o is set, else
// (up to kPagedDecodeCluster ranges) the result.  a.cu null: one row per sequence.
int paged_decode(const PackedArgs& a, cudaStream_t st);
int paged_combine(const PackedArgs& a, int splits, cudaStream_t st);

// paged_decode_q8.cu: the same over 8-bit pages with a scale for each page and kv head, for up to `tiles` tiles of `rows` (8
// or 16) rows per kv head and sequence: in up to kPagedDecodeCluster (a.splits) ranges that a cluster combines, or as a list
// cut into equal parts for all warps.
int paged_decode_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int rows, int tiles,
                    cudaStream_t st);
size_t paged_list_q8_workspace(int batch, int kv_heads, int head_dim, int rows, int tiles);
int paged_list_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int rows, int tiles, void* workspace,
                  cudaStream_t st);
// Every sequence's whole numbers as fp16 pages of 128 keys, `width` of them per sequence (page b * width + w), with their
// table, the lengths (0 for a sequence of more than 128 * width keys) and PackedArgs::key_scale.
int expand_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int width, void* k_out, void* v_out,
              int32_t* table_out, int32_t* lens_out, float2* key_scale, cudaStream_t st);

}  // namespace npub
