// Softmax attention of new tokens over a paged cache, grouped heads of 64 or 128 dims, bf16.
#include "paged.cuh"

namespace {

// One block per row and head; tiles of 128 keys, a thread per key for the scores and a thread per dim for the values. Keys that the row does not
// see are never read.
__global__ void __launch_bounds__(128) attn_paged_rows_kernel(PagedAttnArgs a) {
  __shared__ float q_s[128], p_s[128], red[32];
  __shared__ int page_s[128];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, i = threadIdx.x, D = a.D;
  const int b = paged_seq(a.at, t);
  if (b >= a.at.B) return;
  const int len = a.at.lens[b], pos = len - a.at.starts[b + 1] + (int)t;
  const int64_t head = h / (a.Hq / a.Hkv);
  if (i < D) q_s[i] = __bfloat162float(a.q[(t * a.Hq + h) * D + i]) * a.scale;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t j0 = 0; j0 <= pos && j0 < ((int64_t)a.at.ld << a.at.shift); j0 += 128) {
    __syncthreads();
    const int64_t j = j0 + i;
    const bool seen = j <= pos && (!a.window || j > (int64_t)pos - a.window || j < a.first);
    const int page = seen ? paged_page(a.at, b, (int)(j >> a.at.shift)) : -1;
    page_s[i] = page;
    float s = -INFINITY;
    if (page >= 0) {
      const bf16* k = a.k + ((page * (int64_t)a.Hkv + head) * a.at.page + (j & (a.at.page - 1))) * D;
      s = 0.f;
      for (int d = 0; d < D; d++) s += q_s[d] * __bfloat162float(k[d]);
    }
    const float top = fmaxf(m, block_max(s, red));
    const float c = m == -INFINITY ? 0.f : expf(m - top);
    const float p = page >= 0 && top != -INFINITY ? expf(s - top) : 0.f;
    p_s[i] = p;
    l = l * c + block_sum(p, red);
    __syncthreads();
    if (i < D) {
      o *= c;
      for (int n = 0; n < 128; n++)
        if (page_s[n] >= 0)
          o += p_s[n] * __bfloat162float(a.v[((page_s[n] * (int64_t)a.Hkv + head) * a.at.page + ((j0 + n) & (a.at.page - 1))) * D + i]);
    }
    m = top;
  }
  if (i < D) a.out[(t * a.Hq + h) * D + i] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
}

}  // namespace

int k_attn_paged(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  attn_paged_rows_kernel<<<dim3((unsigned)a.at.T, (unsigned)a.Hq), 128, 0, ctx->stream>>>(a);
  SB_LAUNCHED(ctx);
  return STRICTB200_OK;
}
