// Tokens drawn from logits under temperature, top-k, top-p and min-p, with one given random number per row.
//
// A row's tokens have an order: the larger logit first, of equal ones the lower index. With w = exp((l - max) / temperature) the kept ones are the
// first top_k of that order; of those the shortest beginning whose weight reaches top_p of theirs; of those the ones with w >= min_p. The token is the
// first, by index, at which the running sum of the kept weights exceeds u times their sum.
//
// Weights are whole numbers, w * 2^43 rounded to nearest, from an exponential in 64 bits, and sums of at most 2^20 of them are exact in 64 bits: no
// result depends on the order in which threads add, and a comparison with a sum falls as it does in 64-bit arithmetic except where the two sides agree
// to about 2^-40 of the largest weight.
//
// A row is read from memory once: a cluster of up to eight blocks holds it in shared memory (as ordered keys) and passes over it there. What bounds a row is
// the chain of passes and of meetings of the cluster, two to four microseconds each pair:
//   load, maximum, largest places of 512 groups of threads                                             one meeting
//   top_k of up to 256: the k-th largest of those groups' places bounds the first k tokens from below, and what lies above it, seldom more than
//   a few more, goes to the first block, which ranks them and ends the row alone                       one meeting
// Otherwise, and where that list would be too long:
//   counts (weights) in 1024 bins of (max - l), even in l, and the bin where top_k (top_p) falls       two meetings
//   those in front of and in that bin go to the first block as above, if there are at most LIST        three meetings
//   otherwise the place where the order is cut is found among those of the bin (in the first block if there are at most LIST, by bits of the place where
//   more share the bin), and all blocks sum the kept weights and look for the token
// Batches: two blocks per SM, so that one row's meetings are another's passes.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 1024, LIST = 512;
constexpr int SHARE = 19200;  // keys of a block in shared memory (75 KB, two blocks per SM); the rest of a longer row is read again in every pass
constexpr int MAX_CLUSTER = 8;
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
  const uint32_t b = __float_as_uint(l != l ? -INFINITY : l + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t bits_of_key(uint32_t k) { return k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u); }
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(bits_of_key(k)); }
// A float's bits as a double's: exact for normal numbers, infinities become 2^128 (further than any number), subnormal ones others of no consequence.
__device__ __forceinline__ double wide(uint32_t b) {
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(b << 29));
}
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // of -inf
constexpr uint32_t KEY_INF = 0xFF800000u;

// f * x, f in [0, 1), rounded down, and whether something was lost
__device__ __forceinline__ uint64_t share_of(uint64_t x, float f, bool* lost) {
  const uint64_t g = f >= 1.f ? ~0ull : f > 0.f ? (uint64_t)ldexp((double)f, 64) : 0;
  *lost = x * g != 0;
  return __umul64hi(x, g);
}

struct Shared {
  union {
    struct {
      uint32_t count[BINS];
      uint32_t sum[3][BINS];  // weights in pieces of 15 bits: counters of 32 bits are added to without a loop, and 2^17 members do not overflow them
    } bin;
    struct {
      uint64_t place[LIST], w[LIST], by_rank[LIST];
      uint32_t rank[LIST];
    } list;
  };
  // sums over the cluster of this block's part of the bins (whole for a cluster of one)
  uint32_t part_count[BINS / 2];
  uint64_t part_sum[BINS / 2];
  uint64_t total_count, total_sum;
  uint64_t red[WARPS], red2[WARPS];
  uint64_t pick[6];
  uint64_t best, there, weights, word, drawn;  // what blocks tell one another: largest place, numbers, sums, a cut, the kept weights
  uint32_t n_list;
  long long fraction[64];  // bits of 2^(43 + i / 64)
  uint32_t crest[THREADS];  // largest keys of groups of this block's threads
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_of(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint64_t peer64(const uint64_t* p, int rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peer32(const uint32_t* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}

struct Row {
  Shared& s;
  const uint32_t* keys;  // of the first `held` of this block's `share`
  const void* x;
  int N, f32, first, share, held;
  int blocks, rank, crests;  // crests: groups of this block's threads
  uint32_t top;        // key of the largest logit
  double m, scale, least_d;  // its value, 64 log2(e) / temperature, distance from which on a weight is 0
  float m32, bin_scale;

  // All blocks of the cluster, all threads.
  __device__ __forceinline__ void meet() const {
    __syncthreads();
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __device__ __forceinline__ uint32_t load(int i) const {  // of the block's i-th
    const int64_t at = first + i;
    return key_of(f32 ? ((const float*)x)[at] : __bfloat162float(((const bf16*)x)[at]));
  }
  __device__ __forceinline__ uint32_t key(int i) const { return i < held ? keys[i] : load(i); }
  // the place in the row's order, larger is earlier: the key, then the lower index
  __device__ __forceinline__ uint64_t place(uint32_t k, int i) const { return (uint64_t)k << 20 | (uint32_t)(0xFFFFF - (first + i)); }
  // 2^43 exp((l - max) / T) rounded to a whole number. y = 64 log2(e) (l - max) / T = n + f with n whole and |f| <= 1/2: 2^(y / 64) is 2^(n / 64), from a table of
  // the 64 fractions, times the series of exp(f ln(2) / 64) to the fourth power (off by 4e-14, less than half a unit). The sums that round are additions of a
  // power of two that leaves no bits behind the point.
  // Straight-line, so that several go side by side; keys of -inf are nobody's to ask for.
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    const double d = wide(bits_of_key(k)) - m;
    constexpr double WHOLE = 6755399441055744.0;  // 1.5 * 2^52
    const double t = fma(d, scale, WHOLE), f = fma(d, scale, WHOLE - t);
    const int n = __double2loint(t);
    constexpr double C = 0.69314718055994530942 / 64;
    double p = C * C * C * C / 24;
    p = fma(p, f, C * C * C / 6);
    p = fma(p, f, C * C / 2);
    p = fma(p, f, C);
    p = fma(p, f, 1.0);
    const long long two = s.fraction[n & 63] + ((long long)(n >> 6) << 52);  // 2^(43 + n / 64)
    const uint64_t w = (uint64_t)__double_as_longlong(fma(p, __longlong_as_double(two), 4503599627370496.0)) - 0x4330000000000000ull;
    return d > least_d ? w : 0;  // 2^-45
  }
  // Bins of equal width below the maximum, the last one for all that is further away; never falls with a falling logit.
  __device__ __forceinline__ int bin(uint32_t k) const {
    const float d = (m32 - of_key(k)) * bin_scale;
    return d < (float)(BINS - 1) ? max(0, (int)d) : BINS - 1;
  }
};

__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (WARPS - 1)];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum of v over the threads in front of this one; *all: over all of them.
__device__ __forceinline__ uint64_t block_before64(uint64_t v, uint64_t* red, uint64_t* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = sum;
  __syncthreads();
  uint64_t w = red[lane & (WARPS - 1)];
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *all = __shfl_sync(0xffffffffu, w, WARPS - 1);
  const uint64_t front = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
  return (warp ? front : 0) + sum - v;
}

// f(key, i) for the block's keys from low_key on; four at a time where they are in shared memory.
template <typename F>
__device__ __forceinline__ void each_key(const Row& r, uint32_t low_key, F&& f) {
  const uint4* k4 = (const uint4*)r.keys;
  const int quads = r.held / 4;
#pragma unroll 1
  for (int q = threadIdx.x; q < quads; q += THREADS) {
    const uint4 k = k4[q];
    if (max(max(k.x, k.y), max(k.z, k.w)) < low_key) continue;
    f(k.x, q * 4, k.x >= low_key);
    f(k.y, q * 4 + 1, k.y >= low_key);
    f(k.z, q * 4 + 2, k.z >= low_key);
    f(k.w, q * 4 + 3, k.w >= low_key);
  }
#pragma unroll 1
  for (int i = quads * 4 + threadIdx.x; i < r.share; i += THREADS) {
    const uint32_t k = r.key(i);
    f(k, i, k >= low_key);
  }
}

// The bin where a running sum over the bins (sums: of weights, otherwise of counts) reaches `want`. The first block's list is empty afterwards, and its place free.
struct Crossing {
  int bin;
  uint64_t count;         // members of the bin
  uint64_t front;         // members of the bins in front
  uint64_t want;          // of the bin's own
  bool whole;             // the bin is kept as a whole
};
__device__ __forceinline__ Crossing cross(const Row& r, bool sums, uint64_t want) {
  Shared& s = r.s;
  const int per = BINS / r.blocks;
  if (r.rank == 0 && threadIdx.x == 0) s.n_list = 0;
  r.meet();  // all bins are counted
  const uint32_t* counts = s.bin.count;
  auto sum_of = [&](int i) { return s.bin.sum[0][i] + ((uint64_t)s.bin.sum[1][i] << 15) + ((uint64_t)s.bin.sum[2][i] << 30); };
  int owner = 0;
  uint64_t front_c = 0, front_s = 0;
  if (r.blocks > 1) {
    uint64_t tc = 0, ts = 0;
    for (int i = threadIdx.x; i < per; i += THREADS) {
      uint32_t c[MAX_CLUSTER];
      uint64_t w[MAX_CLUSTER];
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++)
        if (b < r.blocks) {
          c[b] = peer32(&s.bin.count[r.rank * per + i], b);
          if (sums) {
            const int at = r.rank * per + i;
            w[b] = peer32(&s.bin.sum[0][at], b) + ((uint64_t)peer32(&s.bin.sum[1][at], b) << 15) + ((uint64_t)peer32(&s.bin.sum[2][at], b) << 30);
          }
        }
      uint64_t cc = 0, ww = 0;
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++)
        if (b < r.blocks) {
          cc += c[b];
          if (sums) ww += w[b];
        }
      s.part_count[i] = (uint32_t)cc;
      if (sums) s.part_sum[i] = ww;
      tc += cc;
      ts += ww;
    }
    tc = block_sum64(tc, s.red);
    if (sums) ts = block_sum64(ts, s.red2);
    if (threadIdx.x == 0) s.total_count = tc, s.total_sum = ts;
    r.meet();
    uint64_t c[MAX_CLUSTER], w[MAX_CLUSTER];
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++)
      if (b < r.blocks) {
        c[b] = peer64(&s.total_count, b);
        w[b] = sums ? peer64(&s.total_sum, b) : 0;
      }
    owner = r.blocks - 1;
    bool found = false;
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++)
      if (b < r.blocks && !found) {
        if ((sums ? front_s + w[b] : front_c + c[b]) >= want) owner = b, found = true;
        else front_c += c[b], front_s += w[b];
      }
  }
  // the owner's part, two neighbouring bins per thread at most
  uint64_t c2[2] = {0, 0}, w2[2] = {0, 0};
  const int each = (per + THREADS - 1) / THREADS;
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int i = threadIdx.x * each + e;
    if (e < each && i < per) {
      c2[e] = r.blocks > 1 ? peer32(&s.part_count[i], owner) : counts[i];
      if (sums) w2[e] = r.blocks > 1 ? peer64(&s.part_sum[i], owner) : sum_of(i);
    }
  }
  uint64_t all, before_c = front_c + block_before64(c2[0] + c2[1], s.red, &all), before_s = 0;
  if (sums) before_s = front_s + block_before64(w2[0] + w2[1], s.red2, &all);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const uint64_t here = sums ? w2[e] : c2[e], before = sums ? before_s : before_c;
    if (e < each && before < want && before + here >= want) {  // one thread, once
      s.pick[0] = owner * per + threadIdx.x * each + e;
      s.pick[1] = c2[e];
      s.pick[2] = before_c;
      s.pick[3] = want - before;
      s.pick[4] = sums ? c2[e] == 1 : here == want - before;
    }
    before_c += c2[e];
    before_s += w2[e];
  }
  __syncthreads();
  return Crossing{(int)s.pick[0], s.pick[1], s.pick[2], s.pick[3], s.pick[4] != 0};
}

__device__ __forceinline__ void clear_bins(Shared& s, bool sums) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) {
    s.bin.count[i] = 0;
    if (sums) s.bin.sum[0][i] = s.bin.sum[1][i] = s.bin.sum[2][i] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ void add_to_bin(Shared& s, bool sums, int b, uint64_t w) {
  atomicAdd(&s.bin.count[b], 1u);
  if (sums) {
    atomicAdd(&s.bin.sum[0][b], (uint32_t)w & 0x7FFFu);
    atomicAdd(&s.bin.sum[1][b], (uint32_t)(w >> 15) & 0x7FFFu);
    atomicAdd(&s.bin.sum[2][b], (uint32_t)(w >> 30));
  }
}

// The members with keys from low_key on that `of` chooses, from all blocks, into the first block's list, which is empty (at most LIST of them).
template <typename F>
__device__ __forceinline__ void gather(const Row& r, uint32_t low_key, F&& of) {
  Shared& s = r.s;
  auto take = [&](int i, uint32_t k) {
    const uint64_t p = r.place(k, i);
    if (!of(k, p)) return;
    uint32_t at;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(remote(&s.n_list, 0)) : "memory");
    if (at < LIST) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&s.list.place[at], 0)), "l"(p) : "memory");
  };
  each_key(r, low_key, [&](uint32_t k, int i, bool in) {
    if (in) take(i, k);
  });
  r.meet();
}

// Ranks of the list's members (the first block): by_rank. Threads share out the comparisons.
__device__ __forceinline__ void rank_list(Shared& s, int n) {
  for (int i = threadIdx.x; i < n; i += THREADS) s.list.rank[i] = 0;
  __syncthreads();
  int wide = 1;
  while (wide < n) wide <<= 1;
  const int segs = THREADS / min(wide, THREADS), i = threadIdx.x % min(wide, THREADS), seg = threadIdx.x / min(wide, THREADS);
  if (i < n) {
    const uint64_t p = s.list.place[i];
    uint32_t above = 0;
    for (int j = seg; j < n; j += segs) above += s.list.place[j] > p;
    if (above) atomicAdd(&s.list.rank[i], above);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += THREADS) s.list.by_rank[s.list.rank[j]] = s.list.place[j];
  __syncthreads();
}

// Sum over the cluster of every thread's v; slot: a word of each block's that nothing else has used since the last two meetings.
__device__ __forceinline__ uint64_t cluster_sum(const Row& r, uint64_t v, uint64_t* slot) {
  v = block_sum64(v, r.s.red);
  if (r.blocks == 1) return v;
  if (threadIdx.x == 0) *slot = v;
  r.meet();
  uint64_t c[MAX_CLUSTER], sum = 0;
#pragma unroll
  for (int b = 0; b < MAX_CLUSTER; b++)
    if (b < r.blocks) c[b] = peer64(slot, b);
#pragma unroll
  for (int b = 0; b < MAX_CLUSTER; b++)
    if (b < r.blocks) sum += c[b];
  return sum;
}

// The row's end in the first block, from its ranked list: `keep` of it are the kept beginning, or, with want > 0, those up to the weight `want`.
__device__ __forceinline__ void end_row(const Row& r, const DrawArgs& a, int64_t row, int keep, uint64_t want, bool p_of_kept, float top_p, uint64_t least, float u) {
  Shared& s = r.s;
  const int n = min((int)s.n_list, keep), i = threadIdx.x;
  const uint64_t p = i < n ? s.list.by_rank[i] : 0;
  uint64_t w = i < n ? r.weight((uint32_t)(p >> 20)) : 0, all;
  const uint64_t before = block_before64(w, s.red, &all);
  if (p_of_kept) {  // top_p of what top_k kept
    bool lost;
    want = share_of(all, top_p, &lost);
    want += lost;
    if (want < 1) want = 1;
  }
  if (want && before >= want) w = 0;
  if (w < least) w = 0;
  __syncthreads();
  if (i < n) s.list.w[i] = w;
  const uint64_t total = block_sum64(w, s.red2);
  bool lost;
  const uint64_t target = share_of(total, u, &lost);
  if (i == 0) s.pick[0] = 0xFFFFFFFFull;
  // sum of the kept weights up to one's own index
  s.list.place[i] = 0;
  __syncthreads();
  int wide = 1;
  while (wide < n) wide <<= 1;
  const int segs = THREADS / wide, me = i % wide, seg = i / wide;
  if (me < n && s.list.w[me]) {
    const uint32_t mine = (uint32_t)(s.list.by_rank[me] & 0xFFFFF);
    uint64_t sum = 0;
    for (int j = seg; j < n; j += segs)
      if ((uint32_t)(s.list.by_rank[j] & 0xFFFFF) >= mine) sum += s.list.w[j];  // not a higher index: places hold 2^20 - 1 - index
    if (sum) atomicAdd((unsigned long long*)&s.list.place[me], (unsigned long long)sum);
  }
  __syncthreads();
  if (i < n && w && s.list.place[i] > target) atomicMin((unsigned long long*)&s.pick[0], (unsigned long long)(0xFFFFF - (p & 0xFFFFF)));
  __syncthreads();
  if (i < n && w && (0xFFFFF - (p & 0xFFFFF)) == s.pick[0]) {
    a.out[row] = (int32_t)s.pick[0];
    if (a.prob) a.prob[row] = (float)((double)w / (double)total);
  }
}

__global__ void __launch_bounds__(THREADS, 2) draw_kernel(const __grid_constant__ DrawArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *(Shared*)smem;
  uint32_t* keys = (uint32_t*)(smem + (sizeof(Shared) + 15) / 16 * 16);
  pdl_wait();
  pdl_trigger();
  uint32_t rank, blocks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
  const int64_t row = blockIdx.x / blocks;
  const int each = ((a.N + (int)blocks - 1) / (int)blocks + 7) / 8 * 8;
  Row r{s, keys};
  r.x = (const char*)a.x + row * a.ld * (a.f32 ? 4 : 2);
  r.N = a.N;
  r.f32 = a.f32;
  r.blocks = (int)blocks;
  r.rank = (int)rank;
  r.first = min(a.N, (int)rank * each);
  r.share = min(a.N - r.first, each);
  r.held = min(r.share, SHARE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  uint32_t top_key = 0;
  int top_at = 0;
  auto seen = [&](uint32_t k, int i) {  // a thread's indices rise
    if (k > top_key) top_key = k, top_at = i;
  };
  auto take = [&](uint32_t k, int i) {
    if (i < r.held) keys[i] = k;
    seen(k, i);
  };
  if (a.f32 && ((uintptr_t)((const float*)r.x + r.first) & 15) == 0) {
    const float4* x4 = (const float4*)((const float*)r.x + r.first);
    constexpr int AHEAD = 5;  // SHARE / 4 / THREADS is 9.4
    for (int i0 = threadIdx.x; i0 < r.share / 4; i0 += THREADS * AHEAD) {
      float4 v[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; e++)
        if (i0 + e * THREADS < r.share / 4) v[e] = x4[i0 + e * THREADS];
#pragma unroll
      for (int e = 0; e < AHEAD; e++) {
        const int i = (i0 + e * THREADS) * 4;
        if (i0 + e * THREADS < r.share / 4) {
          const uint4 k = make_uint4(key_of(v[e].x), key_of(v[e].y), key_of(v[e].z), key_of(v[e].w));
          if (i + 3 < r.held) *(uint4*)(keys + i) = k;  // SHARE is a multiple of four
          seen(k.x, i);
          seen(k.y, i + 1);
          seen(k.z, i + 2);
          seen(k.w, i + 3);
        }
      }
    }
    for (int i = r.share / 4 * 4 + threadIdx.x; i < r.share; i += THREADS) take(r.load(i), i);
  } else if (!a.f32 && ((uintptr_t)((const bf16*)r.x + r.first) & 15) == 0) {
    const uint4* x8 = (const uint4*)((const bf16*)r.x + r.first);
#pragma unroll 4
    for (int i = threadIdx.x; i < r.share / 8; i += THREADS) {
      const uint4 v = x8[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; e++) take(key_of(__uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16)), i * 8 + e);
    }
    for (int i = r.share / 8 * 8 + threadIdx.x; i < r.share; i += THREADS) take(r.load(i), i);
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < r.share; i += THREADS) take(r.load(i), i);
  }
  uint64_t best = top_key ? r.place(top_key, top_at) : 0;
  // 512 groups in the cluster: threads of a block, or two, four or eight neighbours
  r.crests = THREADS / r.blocks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (o == r.blocks && lane % o == 0) s.crest[threadIdx.x / o] = (uint32_t)(best >> 20);
    const uint64_t v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if (threadIdx.x < 64) s.fraction[threadIdx.x] = __double_as_longlong(exp2(43.0 + threadIdx.x / 64.0));
  if (threadIdx.x == 0) s.n_list = 0;
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  for (int i = 0; i < WARPS; i++) best = s.red[i] > best ? s.red[i] : best;
  if (threadIdx.x == 0) s.best = best;
  r.meet();
  if (r.blocks > 1) {
    uint64_t v[MAX_CLUSTER];
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++) v[b] = b < r.blocks ? peer64(&s.best, b) : 0;
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++) best = v[b] > best ? v[b] : best;
  }
  r.top = (uint32_t)(best >> 20);
  r.m32 = of_key(r.top);
  r.m = wide(bits_of_key(r.top));
  const float heat = a.temperature ? a.temperature[row] : 1.f;
  if (r.top <= KEY_NONE || !(heat > 0.f)) {
    if (rank == 0 && threadIdx.x == 0) {
      a.out[row] = r.top <= KEY_NONE ? -1 : 0xFFFFF - (int)(best & 0xFFFFF);
      if (a.prob) a.prob[row] = r.top <= KEY_NONE ? 0.f : 1.f;
    }
    r.meet();
    return;
  }
  // beside +inf nothing has a weight
  r.scale = r.top >= KEY_INF ? 1e30 : 64 * 1.4426950408889634074 / heat;
  r.least_d = r.scale > 0 ? -2880.0 / r.scale : -1e300;
  r.bin_scale = fminf((BINS - 1) / (32.f * heat), 1e30f);
  if (r.top >= KEY_INF) r.m32 = 3.4028235e38f;  // bins below a largest logit of +inf: that one in the first, whatever is finite by its distance from the largest number
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
  const uint64_t least = min_p > 0.f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * ONE) : 0;
  float u = a.u[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  // Two cuts, top_k's by counts and top_p's by weights, each unless nothing is asked of it. from: lowest place that is kept so far.
  uint64_t from = (uint64_t)(KEY_NONE + 1) << 20, want = 0;
  bool few = false;  // the first block has the kept ones (and some more of the order) in its list, ranked
  bool by_count = false;
#pragma unroll 1
  for (int stage = 0; stage < 2 && !few; stage++) {
    const bool sums = stage == 1;
    by_count = !sums;
    uint32_t low_key = (uint32_t)(from >> 20);
    if (!sums) {
      if (k <= 0 || k >= a.N) continue;
      if (2 * k <= THREADS) {
        // The k-th largest of the groups' largest keys (to 22 bits, downwards) has at least k tokens from it on, and, where the largest are not all in a few
        // groups, not many more.
        const uint32_t mine = r.blocks > 1 ? peer32(&s.crest[threadIdx.x % r.crests], threadIdx.x / r.crests) : s.crest[threadIdx.x];
        uint32_t low = 0;
#pragma unroll 1
        for (uint32_t bit = 1u << 31; bit >= 1u << 10; bit >>= 1)
          if (__syncthreads_count(mine >= (low | bit)) >= k) low |= bit;
        gather(r, max(low, KEY_NONE + 1), [](uint32_t, uint64_t) { return true; });
        few = (r.blocks > 1 ? peer32(&s.n_list, 0) : s.n_list) <= LIST;
        if (few) {
          if (r.rank == 0) rank_list(s, (int)s.n_list);
          break;
        }
        r.meet();  // the number has been read
      }
      uint64_t there = 0;
      each_key(r, KEY_NONE + 1, [&](uint32_t, int, bool in) { there += in; });
      if ((uint64_t)k >= cluster_sum(r, there, &s.there)) continue;  // all that have any weight are kept
      want = k;
    } else {
      if (!(top_p < 1.f)) continue;
      uint64_t sum = 0;
      each_key(r, low_key, [&](uint32_t key, int i, bool in) {
        const uint64_t w = r.weight(key);
        sum += in && r.place(key, i) >= from ? w : 0;
      });
      sum = cluster_sum(r, sum, &s.weights);
      bool lost;
      want = share_of(sum, top_p, &lost);
      want = max((uint64_t)1, want + lost);
      // All weights up to (sum - want) / N together are at most sum - want: the cut is above them, and keys that far down (a thousandth further) stay out of the bins.
      const double tail = (double)(sum - want) / a.N;
      if (tail > 0) {
        const float reach = (float)(heat * log(ONE / tail) * 1.001) + fabsf(r.m32) * 1e-6f;
        if (reach < 1e30f) low_key = max(low_key, key_of(r.m32 - reach));
      }
    }
    int b0 = 0, hi = 52;
    uint64_t known = 0, left = want;
    bool digits = false;  // within bin b0, where more than LIST share it: by the next ten bits of the place
#pragma unroll 1
    while (true) {
      const int lo = max(0, hi - 10), mask = (1 << (hi - lo)) - 1;
      clear_bins(s, sums);
      each_key(r, low_key, [&](uint32_t key, int i, bool in) {
        const uint64_t p = r.place(key, i), w = sums ? r.weight(key) : 0;
        int b = r.bin(key);
        in = in && p >= from;
        if (digits) {
          in = in && b == b0 && (hi == 52 || p >> hi == known);
          b = mask - ((int)(p >> lo) & mask);  // larger digits first
        }
        if (in) add_to_bin(s, sums, b, w);
      });
      const Crossing c = cross(r, sums, left);
      left = c.want;
      if (digits) {
        known = (hi < 52 ? known << (hi - lo) : 0) | (uint64_t)(mask - c.bin);
        hi = lo;
        if (c.whole) {  // all that begin with these bits
          from = max(from, known << hi);
          break;
        }
      } else {
        b0 = c.bin;
        few = c.front + c.count <= LIST;
      }
      if (few || c.count <= LIST) {
        gather(r, low_key, [&](uint32_t key, uint64_t p) {
          const int b = r.bin(key);
          return p >= from && (few ? b <= b0 : b == b0 && (!digits || p >> hi == known));
        });
        if (r.rank == 0) {
          const int n = (int)s.n_list;
          rank_list(s, n);
          if (!few && !sums && threadIdx.x == 0) s.word = s.list.by_rank[left - 1];
          if (!few && sums) {
            uint64_t all;
            const uint64_t w = threadIdx.x < n ? r.weight((uint32_t)(s.list.by_rank[threadIdx.x] >> 20)) : 0, before = block_before64(w, s.red, &all);
            if (before < left && before + w >= left) s.word = s.list.by_rank[threadIdx.x];
          }
        }
        if (few) break;
        r.meet();
        from = max(from, peer64(&s.word, 0));
        break;
      }
      digits = true;
    }
  }
  if (few) {
    if (r.rank == 0) {
      end_row(r, a, row, by_count ? k : LIST, by_count ? 0 : want, by_count && top_p < 1.f, top_p, least, u);
    }
    r.meet();
    return;
  }
  // The draw: a thread sums a contiguous part of the block's share (an odd number of keys, so that a warp's reads meet no bank twice), the sums in front of
  // it tell the one thread whose part holds the token, and its warp looks through that part.
  const int each_thread = (r.share + THREADS - 1) / THREADS | 1, i0 = min(r.share, (int)threadIdx.x * each_thread), i1 = min(r.share, i0 + each_thread);
  const uint32_t from_key = (uint32_t)(from >> 20);
  auto kept = [&](int i) -> uint64_t {
    const uint32_t key = r.key(i);
    if (key < from_key || r.place(key, i) < from) return 0;
    const uint64_t w = r.weight(key);
    return w >= least ? w : 0;
  };
  uint64_t mine = 0, block_total, total = 0;
#pragma unroll 1
  for (int i = i0; i < i1; i += 4) {
    uint32_t key[4];
#pragma unroll
    for (int e = 0; e < 4; e++) key[e] = i + e < i1 ? r.key(i + e) : 0;
    if (max(max(key[0], key[1]), max(key[2], key[3])) < from_key) continue;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint64_t w = r.weight(key[e]);
      mine += key[e] >= from_key && r.place(key[e], i + e) >= from && w >= least ? w : 0;
    }
  }
  uint64_t before = block_before64(mine, s.red, &block_total);
  if (threadIdx.x == 0) s.drawn = block_total;
  r.meet();
  for (int b = 0; b < r.blocks; b++) {
    const uint64_t v = r.blocks > 1 ? peer64(&s.drawn, b) : block_total;
    if (b < r.rank) before += v;
    total += v;
  }
  r.meet();  // nobody leaves while its memory is read
  bool lost;
  const uint64_t target = share_of(total, u, &lost);
  const unsigned mine_it_is = __ballot_sync(0xffffffffu, target >= before && target < before + mine);
  if (!mine_it_is) return;
  const int src = __ffs(mine_it_is) - 1, p0 = __shfl_sync(0xffffffffu, i0, src), p1 = __shfl_sync(0xffffffffu, i1, src);
  before = __shfl_sync(0xffffffffu, before, src);
  for (int i = p0; i < p1; i += 32) {
    const uint64_t w = i + lane < p1 ? kept(i + lane) : 0;
    uint64_t sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + sum > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.out[row] = r.first + i + lane;
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
  const DrawArgs a{x, ld, (int)N, f32, u, temperature, top_p, min_p, top_k, out, prob};
  int blocks = 1;  // of a row: as few as hold it, or eight
  while (blocks < MAX_CLUSTER && N > (int64_t)blocks * SHARE) blocks *= 2;
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)std::min<int64_t>(SHARE, (N + blocks - 1) / blocks + 8) * 4;
  static SbDeviceOnce once;
  SB_CUDA(once.run(ctx->device, [&] { return cudaFuncSetAttribute(draw_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((sizeof(Shared) + 15) / 16 * 16 + SHARE * 4)); }));
  // rows of one launch: as many as the grid takes
  const int64_t most = INT32_MAX / blocks;
  for (int64_t m0 = 0; m0 < M; m0 += most) {
    DrawArgs part = a;
    part.x = (const char*)x + m0 * ld * (f32 ? 4 : 2);
    part.u += m0;
    if (temperature) part.temperature += m0;
    if (top_k) part.top_k += m0;
    if (top_p) part.top_p += m0;
    if (min_p) part.min_p += m0;
    part.out += m0;
    if (prob) part.prob += m0;
    SB_CUDA(sb_launch_cluster(ctx, draw_kernel, dim3((unsigned)(std::min(M - m0, most) * blocks)), dim3(THREADS), smem, dim3((unsigned)blocks), part));
    ctx->launches++;
  }
  return STRICTB200_OK;
}
