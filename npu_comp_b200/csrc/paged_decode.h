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

}  // namespace npub
