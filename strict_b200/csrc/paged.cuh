// What the kernels over a paged cache share: where a row of the packed new tokens belongs, and where a position lies.
#pragma once
#include "common.cuh"

// Keys and values of a layer lie in pages [n_pages, Hkv, page, D]; row b of the table names the pages of sequence b in order. The new tokens of
// all sequences are rows of one packed array: those of sequence b are starts[b] .. starts[b + 1] - 1, the last ones of its lens[b] tokens.
struct PagedView {
  const int32_t* table = nullptr;   // [B, ld]
  const int32_t* lens = nullptr;    // [B]
  const int32_t* starts = nullptr;  // [B + 1]
  int B = 0, ld = 0, n_pages = 0;
  int page = 0, shift = 0;          // slots of a page, a power of two, and its logarithm
  int64_t T = 0;                    // rows of the packed array
};

struct PagedAttnArgs {
  PagedView at;
  const bf16* q = nullptr;  // [T, Hq, D]
  const bf16* k = nullptr;  // pages
  const bf16* v = nullptr;
  int Hq = 0, Hkv = 0, D = 0;
  int window = 0, first = 0;  // a row at position p sees j <= p with j > p - window (0: all) or j < first
  int max_new = 0, max_len = 0;
  float scale = 0.f;
  bf16* out = nullptr;  // [T, Hq, D]
};
int k_attn_paged(strictb200_ctx*, const PagedAttnArgs& a);  // attention_paged.cu

struct PagedRopeArgs {
  PagedView at;
  const bf16* qkv = nullptr;  // [T, (Hq + 2 Hkv) D]
  const float* qgain = nullptr;  // null: no norm
  const float* kgain = nullptr;
  float eps = 0.f, theta = 0.f;
  int Hq = 0, Hkv = 0, D = 0;
  bf16* q_out = nullptr;
  bf16* k = nullptr;
  bf16* v = nullptr;
};
int k_rope_paged(strictb200_ctx*, const PagedRopeArgs& a);  // rope_paged.cu

// Copies page src[i] of every pool over page dst[i]; no page is named twice but as a source. pages.cu
int k_pages_copy(strictb200_ctx*, void* const* pools, int n_pools, int64_t page_bytes, const int32_t* src, const int32_t* dst, int n);

#ifdef __CUDACC__
// Page of slot group `n` of sequence b, or -1 where the table names none.
__device__ __forceinline__ int paged_page(const PagedView& v, int b, int n) {
  if ((unsigned)n >= (unsigned)v.ld) return -1;
  const int p = v.table[(int64_t)b * v.ld + n];
  return p >= 0 && p < v.n_pages ? p : -1;
}
// First position in the window of a row. Rows in front of their sequence (pos < 0) see nothing; counted from there, wide windows would pass 32 bits.
__device__ __forceinline__ int window_begin(int pos, int window) { return window ? max(0, max(pos, 0) - window + 1) : 0; }
// The key tiles (of `kt` positions) that rows up to position hi_pos walk over, the window of whose first one begins at lo_key: those of the first tokens, then those from
// the window on.
struct PagedWalk {
  int first;  // tiles of the first tokens
  int lo;     // tile where the window begins
  int total;
  int end;    // no row sees this position or a later one
  __device__ __forceinline__ int tile(int t) const { return t < first ? t : lo + t - first; }
};
__device__ __forceinline__ PagedWalk paged_walk(const PagedView& v, int len, int lo_key, int hi_pos, int first, int kt) {
  PagedWalk w;
  const int64_t room = min((int64_t)v.ld << v.shift, (int64_t)INT32_MAX - 1024);  // so that a tile's end is an int
  w.end = (int)(room < len ? room : len);
  w.end = max(0, min(w.end, hi_pos + 1));
  const int tiles = (w.end + kt - 1) / kt;
  w.lo = min(lo_key / kt, tiles);
  w.first = min((min(first, w.end) + kt - 1) / kt, w.lo);
  w.total = w.first + tiles - w.lo;
  return w;
}
#endif
