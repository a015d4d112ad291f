// What the kernels of the attention over a paged cache share: the join of their parts.
#pragma once
#include "paged.cuh"
#include "tcgen05.cuh"

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

#ifdef __CUDACC__
// Page numbers of a block's key tiles, fetched by one warp for 32 boxes at a time, the next 32 while the present ones are in use (a look-up per tile
// held a block to a tile per trip to L2). Box i of a tile is in lane i.
struct PageNames {
  int now, next, per;  // tiles of a fetch
  template <typename F>
  __device__ __forceinline__ void begin(int boxes, int lane, F&& page_of) {
    per = 32 / boxes;
    now = page_of(lane / boxes, lane % boxes);
    next = page_of(per + lane / boxes, lane % boxes);
  }
  // of tile i, asked for in order
  template <typename F>
  __device__ __forceinline__ int of(int i, int boxes, int lane, F&& page_of) {
    const int k = i % per;
    if (i && !k) {
      now = next;
      next = page_of(i + per + lane / boxes, lane % boxes);
    }
    const int p = __shfl_sync(0xffffffffu, now, (k * boxes + lane) & 31);
    return lane < boxes ? p : -1;
  }
};
// Which halves of a pair of bf16 are infinities or NaN: bits 15 and 31; and the pair with zeros in their place.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t only_finite(uint32_t w) { return w & ~((not_finite(w) >> 15) * 0xFFFFu); }

// Whether keys [k0, k0 + kn) are all seen by the rows at positions lo_pos .. hi_pos (end: no row sees that position or a later one).
__device__ __forceinline__ bool sees_all(const PagedAttnArgs& a, int end, int k0, int kn, int lo_pos, int hi_pos) {
  return k0 + kn <= end && k0 + kn - 1 <= lo_pos && (!a.window || k0 > hi_pos - a.window || k0 + kn <= a.first);
}

// i-th key tile of a block whose share is every parts-th piece of ct tiles
__device__ __forceinline__ int share_tile(int i, int part, int parts, int ct) { return parts == 1 ? i : (i / ct * parts + part) * ct + i % ct; }
__device__ __forceinline__ int share_count(int total, int part, int parts, int ct) {
  if (parts == 1) return total;
  const int rounds = total / (parts * ct), rest = total - rounds * parts * ct;
  return rounds * ct + min(max(rest - part * ct, 0), ct);
}

// What a weight of zero times a value that is not finite would do to a row that does not see it is avoided by zeros in place of such values in tiles that some
// row does not see whole. Tiles of a block's share where that befell values that some row may see (the i-th ones, some of them more than once; more than
// POISON_TILES: any of the share).
constexpr int POISON_TILES = 24;
struct Poison {
  int n, tile[POISON_TILES];
};
__device__ __forceinline__ void note_poison(Poison& p, int i) {  // one lane of a warp
  const int at = atomicAdd(&p.n, 1);
  if (at < POISON_TILES) p.tile[at] = i;
}
// A row that does see such values gets them here: those of the n tiles i0, i0 + step .. of a block, dims d0 .. d0 + nd - 1 (nd % 4 == 0), added to r. Only groups of
// `grain` keys are gone through that the rows lo_pos .. hi_pos do not see whole, as where the values were replaced: a walk over a whole long sequence would
// hold up a call of 48 us for 1.4 ms at 16000 keys, and with it the other warps of a block that stays. Seldom, so slow. (A weight is positive; that it may have been rounded to zero does
// not matter to the sum: it is not finite either way, and neither does a value that is added twice.)
static __device__ __noinline__ void add_poison(const PagedAttnArgs& a, const PagedWalk& w, int b, int hk, int part, int parts, int ct, int kt, int grain, int lo_pos,
                                               int hi_pos, const Poison& noted, int i0, int step, int n, int pos, int d0, int nd, float* r) {
  const int lo = window_begin(pos, a.window), many = *(volatile const int*)&noted.n;
  const bool any = many > POISON_TILES;
  for (int x = 0; x < (any ? n : many); x++) {
    const int i = any ? i0 + x * step : *(volatile const int*)&noted.tile[x];
    if (i < i0 || (i - i0) % step || (i - i0) / step >= n) continue;  // another stream's
    const int k0 = w.tile(share_tile(i, part, parts, ct)) * kt, end = min(k0 + kt, min(w.end, pos + 1));
    for (int g0 = k0; g0 < end; g0 += grain) {
      bool whole = sees_all(a, w.end, g0, grain, lo_pos, hi_pos);
      for (int j = g0; whole && j < g0 + grain; j += a.at.page) whole = paged_page(a.at, b, j >> a.at.shift) >= 0;
      if (whole) continue;
      for (int j = g0; j < min(g0 + grain, end); j++) {
        if (j < lo && j >= a.first) continue;
        const int page = paged_page(a.at, b, j >> a.at.shift);
        if (page < 0) continue;
        const bf16* v = a.v + ((page * (int64_t)a.Hkv + hk) * a.at.page + (j & (a.at.page - 1))) * a.D + d0;
        for (int d = 0; d < nd; d += 4) {
          const uint2 y = *(const uint2*)(v + d);
          if (!(not_finite(y.x) | not_finite(y.y))) continue;
          for (int e = 0; e < 4; e++) {
            const float z = __bfloat162float(v[d + e]);
            if (!isfinite(z)) r[d + e] += z;
          }
        }
      }
    }
  }
}

// Tensor map of rows of `cols` bf16, boxes of `box` rows x 64 columns, 128-byte swizzle
inline int paged_map_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int box) {
  tc::EncodeFn encode;
  SB_TRY(tc::encode_fn(&encode));
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * 2};
  cuuint32_t boxes[2] = {64u, (cuuint32_t)box};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sb_fail(STRICTB200_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return STRICTB200_OK;
}
#endif
