// Tokens drawn from logits under temperature, top-k, top-p and min-p, with one given random number per row.
//
// A row's tokens have an order: the larger logit first, of equal ones the lower index. With w = exp((l - max) / temperature) the kept ones are the
// first top_k of that order; of those the shortest beginning whose weight reaches top_p of theirs; of those the ones with w >= min_p. The token is the
// first, by index, at which the running sum of the kept weights exceeds u times their sum.
//
// Weights are whole numbers, w * 2^43 rounded to nearest, from an exponential in 64 bits, and sums of at most 2^20 of them are exact in 64 bits: no
// result depends on the order in which threads add, and a comparison with a sum falls as it does in 64-bit arithmetic except where the two sides agree
// to about 2^-40 of the largest weight.
#include "common.cuh"

namespace {

constexpr int THREADS = 1024;
constexpr double ONE = 8796093022208.0;  // 2^43

struct DrawArgs {
  const void* x;
  int64_t ld;
  int N, f32;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* out;
  float* prob;
};

// Larger logits have larger keys; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float l) {
  l = l != l ? -INFINITY : l + 0.f;
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // of -inf

// x * f / 2^64 for f in [0, 1) given as f * 2^64, rounded down, and whether something was lost
__device__ __forceinline__ uint64_t share_of(uint64_t x, float f, bool* lost) {
  const uint64_t g = f >= 1.f ? ~0ull : f > 0.f ? (uint64_t)ldexp((double)f, 64) : 0;
  *lost = x * g != 0;
  return __umul64hi(x, g);
}

struct Row {
  const void* x;
  int N, f32;
  uint32_t top;     // key of the largest logit
  double m, inv_t;  // its value, 1 / temperature
  __device__ __forceinline__ uint32_t key(int i) const {
    return key_of(f32 ? ((const float*)x)[i] : __bfloat162float(((const bf16*)x)[i]));
  }
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    if (k == top) return 1ull << 43;
    if (k <= KEY_NONE || top >= 0xFF800000u) return 0;  // beside +inf nothing has a weight
    return (uint64_t)__double2ll_rn(exp(((double)of_key(k) - m) * inv_t) * ONE);
  }
  // the place in the row's order, larger is earlier: the key, then the lower index
  __device__ __forceinline__ uint64_t place(uint32_t k, int i) const { return (uint64_t)k << 20 | (uint32_t)(0xFFFFF - i); }
};

__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t s = 0;
  for (int i = 0; i < THREADS / 32; i++) s += red[i];
  return s;
}

struct Shared {
  unsigned long long sum[256];
  unsigned count[256];
  uint64_t red[32];
  uint64_t pick[4];
};

// Lowest place that is kept, among the places from `from` on, when the first `want` of them are kept (MASS: the first whose weight in front is below `want`).
template <bool MASS>
__device__ uint64_t lowest_kept(const Row& r, uint64_t from, uint64_t want, Shared& s) {
  uint64_t known = 0;
  int shift = 52;
  while (shift > 0) {
    const int low = shift > 8 ? shift - 8 : 0, bits = shift - low;
    for (int i = threadIdx.x; i < 256; i += THREADS) { s.count[i] = 0; s.sum[i] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < r.N; i += THREADS) {
      const uint32_t k = r.key(i);
      const uint64_t p = r.place(k, i);
      if (p < from || p >> shift != known) continue;
      const int bin = (int)(p >> low) & ((1 << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      if (MASS) atomicAdd(&s.sum[bin], (unsigned long long)r.weight(k));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t above = 0;
      int bin = (1 << bits) - 1;
      for (; bin > 0; bin--) {
        const uint64_t here = MASS ? s.sum[bin] : s.count[bin];
        if (above + here >= want) break;
        above += here;
      }
      const uint64_t here = MASS ? s.sum[bin] : s.count[bin];
      s.pick[0] = bin;
      s.pick[1] = want - above;
      s.pick[2] = MASS ? s.count[bin] <= 1 : here <= want - above;  // all of the bin is kept
    }
    __syncthreads();
    known = known << bits | s.pick[0];
    want = s.pick[1];
    shift = low;
    const bool whole = s.pick[2];
    __syncthreads();
    if (whole) break;
  }
  const uint64_t p = known << shift;
  return p > from ? p : from;
}

__global__ void __launch_bounds__(THREADS) draw_kernel(DrawArgs a) {
  __shared__ Shared s;
  __shared__ uint64_t warp_sums[32];
  const int64_t row = blockIdx.x;
  Row r;
  r.x = (const char*)a.x + row * a.ld * (a.f32 ? 4 : 2);
  r.N = a.N;
  r.f32 = a.f32;
  // the first place of the order
  uint64_t best = 0;
  for (int i = threadIdx.x; i < a.N; i += THREADS) {
    const uint64_t p = r.place(r.key(i), i);
    best = p > best ? p : best;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int i = 0; i < 32; i++) best = s.red[i] > best ? s.red[i] : best;
  r.top = (uint32_t)(best >> 20);
  r.m = of_key(r.top);
  const float heat = a.temperature ? a.temperature[row] : 1.f;
  if (r.top <= KEY_NONE || !(heat > 0.f)) {
    if (threadIdx.x == 0) {
      a.out[row] = r.top <= KEY_NONE ? -1 : 0xFFFFF - (int)(best & 0xFFFFF);
      if (a.prob) a.prob[row] = r.top <= KEY_NONE ? 0.f : 1.f;
    }
    return;
  }
  r.inv_t = 1.0 / heat;
  uint64_t from = (uint64_t)(KEY_NONE + 1) << 20;
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < a.N) from = lowest_kept<false>(r, from, k, s);
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  if (top_p < 1.f) {
    uint64_t sum = 0;
    for (int i = threadIdx.x; i < a.N; i += THREADS) {
      const uint32_t key = r.key(i);
      if (r.place(key, i) >= from) sum += r.weight(key);
    }
    sum = block_sum64(sum, s.red);
    bool lost;
    uint64_t want = share_of(sum, top_p, &lost);
    want += lost;
    if (want < 1) want = 1;
    from = lowest_kept<true>(r, from, want, s);
  }
  const float min_p = a.min_p ? a.min_p[row] : 0.f;
  uint64_t least = min_p > 0.f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * ONE) : 0;
  // the draw: warp w has the w-th contiguous part of the row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = ((a.N + 31) / 32 + 31) / 32 * 32, i0 = warp * part, i1 = min(a.N, i0 + part);
  auto kept = [&](int i) -> uint64_t {
    const uint32_t key = r.key(i);
    if (r.place(key, i) < from) return 0;
    const uint64_t w = r.weight(key);
    return w >= least ? w : 0;
  };
  uint64_t mine = 0;
  for (int i = i0 + lane; i < i1; i += 32) mine += kept(i);
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) warp_sums[warp] = mine;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < 32; i++) {
    if (i < warp) before += warp_sums[i];
    total += warp_sums[i];
  }
  float u = a.u[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  bool lost;
  const uint64_t target = share_of(total, u, &lost);
  if (target < before || target >= before + mine) return;
  for (int i = i0; i < i1; i += 32) {
    const uint64_t w = i + lane < i1 ? kept(i + lane) : 0;
    uint64_t sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + sum > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.out[row] = i + lane;
        if (a.prob) a.prob[row] = (float)((double)w / (double)total);
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}

}  // namespace

int k_draw(strictb200_ctx* ctx, const void* x, int f32, int64_t M, int64_t N, int64_t ld, const float* u, const float* temperature, const int32_t* top_k,
           const float* top_p, const float* min_p, int32_t* out, float* prob) {
  DrawArgs a{x, ld, (int)N, f32, u, temperature, top_p, min_p, top_k, out, prob};
  draw_kernel<<<(unsigned)M, THREADS, 0, ctx->stream>>>(a);
  SB_LAUNCHED(ctx);
  return STRICTB200_OK;
}
