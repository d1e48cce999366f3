// Internal interface of the few-row paged attention and the combination of
// partial results (paged_decode.cu).
#pragma once

#include "fmha_packed.h"

namespace npub {

constexpr int kPagedDecodeRows = 16;  // rows per kv head that paged_decode takes

// Keys [first + s * chunk, first + (s + 1) * chunk) of every sequence for s < splits, partials split0 + s when
// a.part_o is set, else (splits == 1) the result.  a.cu null: one row per sequence.
int paged_decode(const PackedArgs& a, int first, int chunk, int splits, int split0, cudaStream_t st);
int paged_combine(const PackedArgs& a, int splits, cudaStream_t st);

}  // namespace npub
