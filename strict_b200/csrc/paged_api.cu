// C entry points of the paged cache's operators and of the filtered draw.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "paged.cuh"

namespace {

// The arguments are looked at before the context is touched, so that a refusal needs no GPU.
#define PAGED_CONTEXT(ctx) \
  if (!(ctx)) return sb_fail(STRICTB200_ERR_INVALID_ARG, "null context")

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }
bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// The checks that every operator over a paged cache makes, and its view of the cache.
int paged_view(PagedView* v, const int32_t* table, const int32_t* lens, const int32_t* starts, int B, int64_t T, int n_pages, int page, int table_ld) {
  SB_REQUIRE(B >= 0 && T >= 0 && T <= (1 << 30), "bad shape: B, T not negative, T at most 2^30");
  SB_REQUIRE(n_pages > 0 && table_ld > 0, "bad shape: n_pages and table_ld must be positive");
  if (page < 16 || page > 256 || (page & (page - 1))) return sb_fail(STRICTB200_ERR_UNSUPPORTED, "pages hold 16, 32, 64, 128 or 256 positions");
  if (B && T) SB_REQUIRE(table && lens && starts, "null pointer");
  SB_REQUIRE(aligned4(table) && aligned4(lens) && aligned4(starts), "table, lens and starts must be aligned to their type");
  int shift = 4;
  while ((1 << shift) < page) shift++;
  *v = PagedView{table, lens, starts, B, table_ld, n_pages, page, shift, T};
  return STRICTB200_OK;
}
int paged_heads(int Hq, int Hkv, int D, int n_pages, int page) {
  if (D != 64 && D != 128) return sb_fail(STRICTB200_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  SB_REQUIRE(Hq > 0 && Hkv > 0, "bad shape: no heads");
  // positions of all pages and heads are rows of one matrix, with 32-bit coordinates
  if (Hq > 65535 || Hkv > 65535 || (int64_t)n_pages * Hkv * page > INT32_MAX)
    return sb_fail(STRICTB200_ERR_UNSUPPORTED, "more than 65535 heads, or than 2^31 - 1 positions of all pages and heads");
  return STRICTB200_OK;
}

}  // namespace

extern "C" {

int strictb200_attn_paged(strictb200_ctx* ctx, const uint16_t* q, const uint16_t* kpages, const uint16_t* vpages, const int32_t* table, const int32_t* lens,
                          const int32_t* starts, int B, int64_t T, int max_new, int max_len, int Hq, int Hkv, int D, int n_pages, int page, int table_ld,
                          int window, int first, float scale, uint16_t* out) {
  PAGED_CONTEXT(ctx);
  PagedAttnArgs a;
  SB_TRY(paged_heads(Hq, Hkv, D, n_pages, page));
  SB_REQUIRE(Hq % Hkv == 0, "Hq must be a multiple of Hkv");
  if (Hq / Hkv > 128) return sb_fail(STRICTB200_ERR_UNSUPPORTED, "at most 128 query heads per key/value head");
  SB_REQUIRE(max_new >= 0 && max_len >= 0 && window >= 0 && first >= 0, "max_new, max_len, window and first must not be negative");
  SB_REQUIRE(scale > 0.f && std::isfinite(scale), "scale must be positive and finite");
  SB_TRY(paged_view(&a.at, table, lens, starts, B, T, n_pages, page, table_ld));
  if (!B || !T) return STRICTB200_OK;
  SB_REQUIRE(q && kpages && vpages && out, "null pointer");
  SB_REQUIRE(aligned16(q) && aligned16(kpages) && aligned16(vpages) && aligned16(out), "q, pages and out must be 16-byte aligned");
  const uint64_t rows = (uint64_t)T * Hq * D * 2, pages = (uint64_t)n_pages * Hkv * page * D * 2;
  SB_REQUIRE(out == q || !overlap(out, rows, q, rows), "out overlaps q without being it");  // a row's place in the one is another row's in the other
  SB_REQUIRE(!overlap(out, rows, kpages, pages) && !overlap(out, rows, vpages, pages), "out overlaps the pages");
  a.q = (const bf16*)q; a.k = (const bf16*)kpages; a.v = (const bf16*)vpages; a.out = (bf16*)out;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.window = window; a.first = first; a.max_new = max_new; a.max_len = max_len; a.scale = scale;
  SB_ENTER(ctx);
  return k_attn_paged(ctx, a);
}

int strictb200_rope_qknorm_paged(strictb200_ctx* ctx, const uint16_t* qkv, const int32_t* table, const int32_t* lens, const int32_t* starts, int B, int64_t T,
                                 int Hq, int Hkv, int D, const float* qgain, const float* kgain, float eps, float theta, int n_pages, int page, int table_ld,
                                 uint16_t* q_out, uint16_t* kpages, uint16_t* vpages) {
  PAGED_CONTEXT(ctx);
  PagedRopeArgs a;
  SB_TRY(paged_heads(Hq, Hkv, D, n_pages, page));
  SB_REQUIRE(theta > 0.f && std::isfinite(theta) && eps >= 0.f, "theta must be positive and finite, eps not negative");
  SB_TRY(paged_view(&a.at, table, lens, starts, B, T, n_pages, page, table_ld));
  if (!B || !T) return STRICTB200_OK;
  SB_REQUIRE(qkv && q_out && kpages && vpages, "null pointer");
  SB_REQUIRE(!qgain == !kgain, "gains for both queries and keys, or for neither");
  SB_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(kpages) && aligned16(vpages) && aligned16(qgain) && aligned16(kgain),
             "rows, gains and pages must be 16-byte aligned");
  const uint64_t in = (uint64_t)T * (Hq + 2 * (uint64_t)Hkv) * D * 2, rows = (uint64_t)T * Hq * D * 2;
  SB_REQUIRE(!overlap(q_out, rows, qkv, in), "q_out overlaps qkv");  // a row's place in the one is another row's in the other
  a.qkv = (const bf16*)qkv; a.qgain = qgain; a.kgain = kgain; a.eps = eps; a.theta = theta; a.Hq = Hq; a.Hkv = Hkv; a.D = D;
  a.q_out = (bf16*)q_out; a.k = (bf16*)kpages; a.v = (bf16*)vpages;
  SB_ENTER(ctx);
  return k_rope_paged(ctx, a);
}

int strictb200_pages_copy(strictb200_ctx* ctx, void* const* pools, int n_pools, int n_pages, int64_t page_bytes, const int32_t* src, const int32_t* dst, int n) {
  PAGED_CONTEXT(ctx);
  SB_REQUIRE(n_pools >= 0 && n >= 0 && n_pages >= 0, "negative size");
  SB_REQUIRE(page_bytes > 0 && page_bytes % 16 == 0 && page_bytes <= ((int64_t)1 << 40), "page_bytes must be a positive multiple of 16, at most 2^40");
  if (!n || !n_pools) return STRICTB200_OK;
  SB_REQUIRE(pools && src && dst, "null pointer");
  for (int i = 0; i < n_pools; i++) SB_REQUIRE(pools[i] && aligned16(pools[i]), "pools must be 16-byte aligned device arrays");
  for (int i = 0; i < n; i++) SB_REQUIRE(src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages, "page number out of range");
  try {  // all copies happen at once: a page that is written is neither read nor written by another copy
    std::vector<int32_t> s(src, src + n), d(dst, dst + n);
    std::sort(s.begin(), s.end());
    std::sort(d.begin(), d.end());
    for (int i = 0, j = 0; i < n; i++) {
      SB_REQUIRE(!i || d[i] != d[i - 1], "a page is the destination of two copies");
      while (j < n && s[j] < d[i]) j++;
      SB_REQUIRE(j == n || s[j] != d[i], "a page is both source and destination");
    }
  } catch (const std::bad_alloc&) {
    return sb_fail(STRICTB200_ERR_OOM, "pages_copy: no host memory for the page numbers");
  }
  SB_ENTER(ctx);
  return k_pages_copy(ctx, pools, n_pools, page_bytes, src, dst, n);
}

int strictb200_sample(strictb200_ctx* ctx, const void* logits, int dtype, int64_t M, int64_t N, int64_t ld, const float* u, const float* temperature,
                      const int32_t* top_k, const float* top_p, const float* min_p, int32_t* out, float* prob) {
  PAGED_CONTEXT(ctx);
  SB_REQUIRE(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  SB_REQUIRE(M >= 0 && M <= INT32_MAX && N > 0 && ld >= N, "bad shape (ld must be at least N)");
  if (N > (1 << 20)) return sb_fail(STRICTB200_ERR_UNSUPPORTED, "at most 2^20 tokens");
  if (!M) return STRICTB200_OK;
  SB_REQUIRE(logits && u && out, "null pointer");
  SB_REQUIRE(((uintptr_t)logits & (dtype ? 3 : 1)) == 0, "logits must be aligned to their type");
  SB_REQUIRE(aligned4(u) && aligned4(temperature) && aligned4(top_k) && aligned4(top_p) && aligned4(min_p) && aligned4(out) && aligned4(prob),
             "arrays of a value per row must be aligned to their type");
  const uint64_t row_bytes = (uint64_t)M * 4, bytes = ((uint64_t)(M - 1) * ld + N) * (dtype ? 4 : 2);
  SB_REQUIRE(!overlap(out, row_bytes, logits, bytes) && !(prob && (overlap(prob, row_bytes, logits, bytes) || overlap(prob, row_bytes, out, row_bytes))),
             "out and prob overlap neither the logits nor one another");
  SB_ENTER(ctx);
  return k_draw(ctx, logits, dtype, M, N, ld, u, temperature, top_k, top_p, min_p, out, prob);
}

}  // extern "C"
