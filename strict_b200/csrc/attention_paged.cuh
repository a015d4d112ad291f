// What the kernels of the attention over a paged cache share: the join of their parts.
#pragma once
#include "paged.cuh"

// Unnormalised outputs of rows whose keys were split, [T, Hq, parts]; an output is read only where its sum is not zero.
struct PagedJoin {
  float* o = nullptr;    // [.., D]
  float2* ml = nullptr;  // running maximum (log2) and sum relative to it
  int parts = 0;
};
int paged_join_scratch(strictb200_ctx*, const PagedAttnArgs& a, int parts, PagedJoin* join);
int paged_join(strictb200_ctx*, const PagedAttnArgs& a, const PagedJoin& join);
int64_t paged_walk_tiles(const PagedAttnArgs& a, int kt);  // tiles of kt keys that the rows of a sequence of max_len tokens walk over
int k_attn_paged_tiles(strictb200_ctx*, const PagedAttnArgs& a);  // attention_paged_tc.cu
