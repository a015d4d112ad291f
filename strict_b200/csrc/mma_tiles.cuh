// Pieces of the kernels that feed mma.sync m16n8k16 (bf16) from shared-memory tiles of 64 or 128 dims per row, filled by cp.async.
#pragma once
#include "common.cuh"

#ifdef __CUDACC__
namespace mt {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t s, const void* g, bool valid) {
  int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(g), "r"(sz));
}
__device__ __forceinline__ void cp_async16_hint(uint32_t s, const void* g, bool valid, uint64_t policy) {
  int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;\n" ::"r"(s), "l"(g), "r"(sz), "l"(policy));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return f32_to_bf16_bits(lo) | (f32_to_bf16_bits(hi) << 16);
}
// The softmax weights enter the P.V product as two bf16 terms, p = hi + lo (16 mantissa bits):
// a single bf16 P is off by up to 2^-9, which is enough to move the bf16-rounded attention
// output by an ulp on a few percent of its elements, and the E4M3 quantisation that follows
// turns each such ulp into a 6-12 % step. V is exact in bf16, so two MMAs recover the product.
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t& hi, uint32_t& lo) {
  float ah = round_bf16(a), bh = round_bf16(b);
  hi = pack_bf16(ah, bh);
  lo = pack_bf16(a - ah, b - bh);
}
// HD = dims of a row (64 or 128): rows of HD / 8 chunks of 16 bytes, chunk c of row r at chunk c ^ (r & 7)
template <int HD = 128>
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) { return (uint32_t)(row * 2 * HD + ((chunk ^ (row & 7)) << 4)); }

}  // namespace mt
#endif
