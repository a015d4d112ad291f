// Copies of cache pages.
#include <algorithm>

#include "paged.cuh"

namespace {

// Pools and pairs of one launch, in its parameters (4 KB): nothing to stage, nothing that a later call could overwrite, and a recorded launch keeps them.
constexpr int COPY_POOLS = 96, COPY_PAIRS = 400;
struct CopyArgs {
  uint4* pool[COPY_POOLS];
  int2 pair[COPY_PAIRS];
  int64_t vecs;  // 16-byte words of a page
};

// grid (pieces of a page, pairs, pools)
__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ CopyArgs a) {
  const int2 p = a.pair[blockIdx.y];
  uint4* pool = a.pool[blockIdx.z];
  const uint4* src = pool + p.x * a.vecs;
  uint4* dst = pool + p.y * a.vecs;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.vecs; i += (int64_t)gridDim.x * 256) dst[i] = src[i];
}

}  // namespace

int k_pages_copy(strictb200_ctx* ctx, void* const* pools, int n_pools, int64_t page_bytes, const int32_t* src, const int32_t* dst, int n) {
  CopyArgs a;
  a.vecs = page_bytes / 16;
  const int64_t pieces = std::min<int64_t>((a.vecs + 1023) / 1024, 65535);
  for (int i0 = 0; i0 < n; i0 += COPY_PAIRS) {
    const int pairs = std::min(n - i0, COPY_PAIRS);
    for (int i = 0; i < pairs; i++) a.pair[i] = make_int2(src[i0 + i], dst[i0 + i]);
    for (int p0 = 0; p0 < n_pools; p0 += COPY_POOLS) {
      const int np = std::min(n_pools - p0, COPY_POOLS);
      for (int p = 0; p < np; p++) a.pool[p] = (uint4*)pools[p0 + p];
      pages_copy_kernel<<<dim3((unsigned)pieces, (unsigned)pairs, (unsigned)np), 256, 0, ctx->stream>>>(a);
      SB_LAUNCHED(ctx);
    }
  }
  return STRICTB200_OK;
}
