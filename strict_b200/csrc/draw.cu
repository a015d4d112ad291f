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
// A row is read from memory once: a cluster of up to eight blocks holds it in shared memory and passes over it there. What bounds a row is
// the chain of passes and of meetings of the cluster, two to four microseconds each pair:
//   load, maximum, largest places of 512 groups of threads                                             one meeting
//   top_k of up to 256: the k-th largest of those groups' places bounds the first k tokens from below, and what lies above it, seldom more than
//   a few more, goes to the first block, which ranks them and ends the row alone                       one meeting
// Otherwise, and where that list would be too long:
//   counts (weights) in 1024 bins of (max - l), even in l, and the bin where top_k (top_p) falls       two meetings
//   those in front of and in that bin go to the first block as above, if there are at most LIST        three meetings
//   otherwise the place where the order is cut is found among those of the bin (in the first block if there are at most LIST, by bits of the place where
//   more share the bin), and all blocks sum the kept weights and look for the token
// Many rows: a block per row, which keeps a part of it and reads the rest again from L2 in every pass; the instructions of an SM's row bound it (256 rows of 151936: 37 us
// greedy, 77 with top_k 20, 107 unfiltered, 270 to 400 with a top_p of 0.9 over flat logits; one row 7.4, 13.4, 13.4, 42 to 57). A row with a top_p that no short list holds
// takes 160 us on its SM, 75 or 148 of them as long as one, and with mixed wishes (170 us) such a row is the launch: most other SMs are done before it.
// Times here and below: calls in a row on the same logits.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int GROUPS = 512;  // of threads of a cluster, whose largest keys bound the first of the order
constexpr int BINS = 1024, LIST = 512;
constexpr int PIECE = 128;  // quads of logits that a warp sums at a time for the draw
// Keys of a block in shared memory: 75 KB where two blocks share an SM, 186 KB where one has it; the rest of a longer share is read again in every pass.
template <int THREADS>
constexpr int share_kept() { return THREADS == 512 ? 19072 : 47488; }
constexpr int MAX_CLUSTER = 8;
constexpr double ONE = 8796093022208.0;  // 2^43

}  // namespace

// What a row's top_k cuts to: 0 where it is off, below 1 or from N on.
__host__ __device__ int sb_draw_top_k(int wish, int N) { return wish > 0 && wish < N ? wish : 0; }
// Whether the first k tokens are looked for in a list before there are bins: half as many as there are groups, so that seldom more come with them than it takes.
__host__ __device__ bool sb_draw_lists(int k) { return k > 0 && k <= GROUPS / 2; }

// How far below the largest logit a row's logits may stay out of the bins where the order is cut at the weight `want` of `sum`. What is left out
// together weighs sum - want at most: whole numbers none of which is above k = floor((sum - want) / N). That is what weights become that are below k + 1/2 before
// they are rounded, so it is the distance of that weight, and a thousandth more, far above what a weight, this result and its difference from the largest logit
// are off by. (From a k of 2^43 (1 - 4e-11) on a thousandth is less than that, but then `want` is below 2^43, which the largest logit has alone.)
__host__ __device__ float sb_draw_reach(uint64_t sum, uint64_t want, int N, float heat, float top) {
  const double bound = (double)((sum - want) / (uint64_t)N) + 0.5;
  return (float)(heat * log(ONE / bound) * 1.001) + fabsf(top) * 1e-6f;
}

namespace {

struct DrawArgs {
  const void* x;
  int64_t ld;
  int N, f32;
  int M;  // rows, where their order may change
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* out;
  float* prob;
};

// Larger logits have larger keys; -0 counts as 0. NaN counts as -inf: it is left out by every comparison and has no key.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u)); }
__device__ __forceinline__ float of_place(uint64_t p) { return of_key((uint32_t)(p >> 20)); }
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // of -inf
constexpr float LEAST = -3.402823466e38f;  // of the logits that can be drawn

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
      uint64_t sum[BINS];
    } bin;
    struct {
      uint64_t place[LIST], by_rank[LIST];
    } list;
    uint64_t piece_sum[(1 << 20) / (4 * PIECE)];  // of the draw's pieces of the longest share
  };
  // sums over the cluster of this block's part of the bins (whole for a cluster of one)
  uint32_t part_count[BINS / 2];
  uint64_t part_sum[BINS / 2];
  uint64_t total_count, total_sum;
  uint64_t red[32], red2[32];
  uint64_t pick[4];
  uint64_t best, there, weights, word, drawn;  // what blocks tell one another: largest place, numbers, sums, a cut, the kept weights
  uint32_t n_list;
  long long fraction[64 * 8];  // bits of 2^(43 + i / 64), eight copies side by side: neighbouring lanes read other banks
  uint32_t crest[GROUPS];  // largest keys of groups of this block's threads
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
  const float* near;  // the first `held` of this block's `share` of the logits
  const void* x;
  int f32, vec, first, share, held;  // vec: rows begin at 16 bytes
  int blocks, rank, crests;  // crests: groups of this block's threads
  double m, scale;  // the largest logit, 64 log2(e) / temperature
  float m32, bin_scale, least_l, zero_l;  // least_l: from here on a weight is not 0 (2^-45 of the largest); zero_l: a little below
  bool plain;  // zero_l is near enough, and the largest logit is finite

  // All blocks of the cluster, all threads.
  __device__ __forceinline__ void meet() const {
    __syncthreads();
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __device__ __forceinline__ float load(int i) const {  // the block's i-th logit
    const int64_t at = first + i;
    return f32 ? ((const float*)x)[at] : __bfloat162float(((const bf16*)x)[at]);
  }
  // Four logits from 4 q on, from memory (-inf behind the share), and from wherever they are.
  __device__ __forceinline__ float4 far(int q) const {
    const int i = q * 4;
    if (vec && i + 3 < share) {
      if (f32) return *(const float4*)((const float*)x + first + i);
      const uint2 v = *(const uint2*)((const bf16*)x + first + i);
      return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
    }
    return make_float4(i < share ? load(i) : -INFINITY, i + 1 < share ? load(i + 1) : -INFINITY, i + 2 < share ? load(i + 2) : -INFINITY,
                       i + 3 < share ? load(i + 3) : -INFINITY);
  }
  __device__ __forceinline__ float4 quad(int q) const { return q < held / 4 ? ((const float4*)near)[q] : far(q); }
  // the place in the row's order, larger is earlier: the key, then the lower index
  __device__ __forceinline__ uint64_t place(float l, int i) const { return (uint64_t)key_of(l) << 20 | (uint32_t)(0xFFFFF - (first + i)); }
  // 2^43 exp((l - max) / T) rounded to a whole number. y = 64 log2(e) (l - max) / T = n + f with n whole and |f| <= 1/2: 2^(y / 64) is 2^(n / 64), from a table of
  // the 64 fractions, times the series of exp(f ln(2) / 64) to the fourth power (off by 4e-14 of the weight, a third of a unit at most). The sums that
  // round are additions of a power of two that leaves no bits behind the point. Straight-line, so that several go side by side.
  // This is of a logit as a 64-bit number, exactly (heats may be as small as the least numbers are), with the bias of that addition; neither far away nor above the largest.
  static constexpr uint64_t BIAS = 0x4330000000000000ull;
  __device__ __forceinline__ uint64_t weight_of(double x) const {
    const double d = x - m;
    constexpr double WHOLE = 6755399441055744.0;  // 1.5 * 2^52
    const double t = fma(d, scale, WHOLE), f = fma(d, scale, WHOLE - t);
    const int n = __double2loint(t);
    constexpr double C = 0.69314718055994530942 / 64;
    double p = C * C * C * C / 24;
    p = fma(p, f, C * C * C / 6);
    p = fma(p, f, C * C / 2);
    p = fma(p, f, C);
    p = fma(p, f, 1.0);
    const long long two = s.fraction[(n & 63) << 3 | (threadIdx.x & 7)] + ((long long)(n >> 6) << 52);  // 2^(43 + n / 64)
    return (uint64_t)__double_as_longlong(fma(p, __longlong_as_double(two), 4503599627370496.0));
  }
  __device__ __forceinline__ uint64_t weight(float l) const {  // of any logit
    const uint64_t w = weight_of((double)fminf(l, -LEAST)) - BIAS;  // +inf as the largest number, which `m` is beside it
    return l >= least_l ? w : 0;
  }
  // The weights of four logits from `cut` on together, where `plain`: what is below counts as zero_l, whose weight is 0. (With a choice behind each weight, and
  // a place in the order to compare: 67 instructions a logit for a row without filters, 45 this
  // way: 256 rows 139 us and 105.)
  __device__ __forceinline__ uint64_t weights(const float4& v, float cut) const {
    if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut)) return 0;
    return weight_of(v.x >= cut ? v.x : zero_l) + weight_of(v.y >= cut ? v.y : zero_l) + weight_of(v.z >= cut ? v.z : zero_l) +
           weight_of(v.w >= cut ? v.w : zero_l) - 4 * BIAS;
  }
  // Bins of equal width below the maximum, the last one for all that is further away; never falls with a falling logit.
  __device__ __forceinline__ int bin(float l) const {
    const float d = (m32 - l) * bin_scale;
    return d < (float)(BINS - 1) ? max(0, (int)d) : BINS - 1;
  }
};

template <int THREADS>
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & ((THREADS / 32) - 1)];
#pragma unroll
  for (int o = (THREADS / 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum of v over the threads in front of this one; *all: over all of them.
template <int THREADS>
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
  uint64_t w = red[lane & ((THREADS / 32) - 1)];
#pragma unroll
  for (int o = 1; o < (THREADS / 32); o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *all = __shfl_sync(0xffffffffu, w, (THREADS / 32) - 1);
  const uint64_t front = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
  return (warp ? front : 0) + sum - v;
}

// f(l, i, l >= low) for the block's logits, four at a time (-inf behind the last); not for four that are all below.
template <int THREADS, typename F>
__device__ __forceinline__ void each(const Row& r, float low, F&& f) {
  auto four = [&](const float4& v, int q) {
    if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= low)) return;
    f(v.x, q * 4, v.x >= low);
    f(v.y, q * 4 + 1, v.y >= low);
    f(v.z, q * 4 + 2, v.z >= low);
    f(v.w, q * 4 + 3, v.w >= low);
  };
  const int near = r.held / 4, all = (r.share + 3) / 4;
#pragma unroll 1
  for (int q = threadIdx.x; q < near; q += THREADS) four(((const float4*)r.near)[q], q);
#pragma unroll 1
  for (int q = near + threadIdx.x; q < all; q += 2 * THREADS) {  // two requests on their way
    const float4 v0 = r.far(q), v1 = r.far(q + THREADS);
    four(v0, q);
    four(v1, q + THREADS);
  }
}

// The bin where a running sum over the bins (sums: of weights, otherwise of counts) reaches `want`. The first block's list is empty afterwards, and its place free.
struct Crossing {
  int bin;
  uint64_t count;         // members of the bin; 0: the sum of all bins is less, for all blocks alike, and the rest is undefined
  uint64_t front;         // members of the bins in front
  uint64_t want;          // of the bin's own
};
template <int THREADS>
__device__ __forceinline__ Crossing cross(const Row& r, bool sums, uint64_t want) {
  Shared& s = r.s;
  const int per = BINS / r.blocks;
  if (r.rank == 0 && threadIdx.x == 0) s.n_list = 0;
  r.meet();  // all bins are counted
  const uint32_t* counts = s.bin.count;
  int owner = 0;
  uint64_t front_c = 0, front_s = 0;
  if (r.blocks > 1) {
    uint64_t tc = 0, ts = 0;
    // the threads of a bin (THREADS / per of them, one or more neighbours) read from every that-many-th block
    const int readers = THREADS / per, i = threadIdx.x / readers;
    uint32_t cc = 0;
    uint64_t ww = 0;
    for (int b = threadIdx.x % readers; b < r.blocks; b += readers) {
      const int at = r.rank * per + i;
      const uint32_t c0 = peer32(&s.bin.count[at], b);
      if (sums) {
        ww += peer64(&s.bin.sum[at], b);
      }
      cc += c0;
    }
    for (int o = 1; o < readers; o <<= 1) {
      cc += __shfl_xor_sync(0xffffffffu, cc, o);
      if (sums) ww += __shfl_xor_sync(0xffffffffu, ww, o);
    }
    if (threadIdx.x % readers == 0) {
      s.part_count[i] = cc;
      if (sums) s.part_sum[i] = ww;
      tc = cc;
      ts = ww;
    }
    tc = block_sum64<THREADS>(tc, s.red);
    if (sums) ts = block_sum64<THREADS>(ts, s.red2);
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
      if (sums) w2[e] = r.blocks > 1 ? peer64(&s.part_sum[i], owner) : s.bin.sum[i];
    }
  }
  uint64_t all, before_c = front_c + block_before64<THREADS>(c2[0] + c2[1], s.red, &all), before_s = 0;
  if (sums) before_s = front_s + block_before64<THREADS>(w2[0] + w2[1], s.red2, &all);
  if (threadIdx.x == 0) s.pick[1] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const uint64_t here = sums ? w2[e] : c2[e], before = sums ? before_s : before_c;
    if (e < each && before < want && before + here >= want) {  // one thread, once
      s.pick[0] = owner * per + threadIdx.x * each + e;
      s.pick[1] = c2[e];
      s.pick[2] = before_c;
      s.pick[3] = want - before;
    }
    before_c += c2[e];
    before_s += w2[e];
  }
  __syncthreads();
  return Crossing{(int)s.pick[0], s.pick[1], s.pick[2], s.pick[3]};
}

template <int THREADS>
__device__ __forceinline__ void clear_bins(Shared& s, bool sums) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) {
    s.bin.count[i] = 0;
    if (sums) s.bin.sum[i] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ void add_to_bin(Shared& s, bool sums, int b, uint64_t w) {
  atomicAdd(&s.bin.count[b], 1u);
  if (sums) {  // in halves, the carry by what the lower one held: an addition of 64 bits is a loop here
    uint32_t* half = (uint32_t*)&s.bin.sum[b];
    const uint32_t lo = (uint32_t)w, old = atomicAdd(half, lo);
    atomicAdd(half + 1, (uint32_t)(w >> 32) + (old + lo < lo));
  }
}

// The logits from `low` to `high` that `of` chooses, from all blocks, into the first block's list, which is empty (at most LIST of them).
template <int THREADS, typename F>
__device__ __forceinline__ void gather(const Row& r, float low, float high, F&& of) {
  Shared& s = r.s;
  auto take = [&](float l, int i) {
    if (!(l >= low && l <= high)) return;
    const uint64_t p = r.place(l, i);
    if (!of(l, p)) return;
    uint32_t at;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(remote(&s.n_list, 0)) : "memory");
    if (at < LIST) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&s.list.place[at], 0)), "l"(p) : "memory");
  };
  auto four = [&](const float4& v, int q) {
    if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= low)) return;
    take(v.x, q * 4);
    take(v.y, q * 4 + 1);
    take(v.z, q * 4 + 2);
    take(v.w, q * 4 + 3);
  };
  const int near = r.held / 4, all = (r.share + 3) / 4;
#pragma unroll 1
  for (int q = threadIdx.x; q < near; q += THREADS) four(((const float4*)r.near)[q], q);
#pragma unroll 1
  for (int q = near + threadIdx.x; q < all; q += 2 * THREADS) {
    const float4 v0 = r.far(q), v1 = r.far(q + THREADS);
    four(v0, q);
    four(v1, q + THREADS);
  }
  r.meet();
}

// Values of threads 0 .. n - 1 in falling order (a bitonic network over the next power of two; the others hold 0 and get what is left): thread i's is returned.
// Steps between lanes by shuffles, between warps through `line` (LIST values). All threads of the block.
template <int THREADS>
__device__ __forceinline__ uint64_t sorted(uint64_t v, int n, uint64_t* line) {
  const int i = threadIdx.x;
  int wide = 2;
  while (wide < n) wide <<= 1;
#pragma unroll 1
  for (int size = 2; size <= wide; size <<= 1)
#pragma unroll 1
    for (int step = size >> 1; step > 0; step >>= 1) {
      uint64_t other;
      if (step >= 32) {
        __syncthreads();
        if (i < LIST) line[i] = v;
        __syncthreads();
        other = i < LIST ? line[i ^ step] : 0;
      } else {
        other = __shfl_xor_sync(0xffffffffu, v, step);
      }
      const bool larger = ((i & size) == 0) == ((i & step) == 0);  // this end of the pair keeps the larger
      v = larger == (v > other) ? v : other;
    }
  __syncthreads();
  return v;
}

// The list's members (the first block) in the order of their places: by_rank.
template <int THREADS>
__device__ __forceinline__ void rank_list(Shared& s, int n) {
  const int i = threadIdx.x;
  const uint64_t p = sorted<THREADS>(i < n ? s.list.place[i] : 0, n, s.list.by_rank);
  if (i < LIST) s.list.by_rank[i] = p;
  __syncthreads();
}

// The k-th largest of the groups' largest keys (to 22 bits, downwards) has at least k tokens from it on, and, where the largest are not all in a few
// groups, not many more.
template <int THREADS>
__device__ __forceinline__ float crest_bound(const Row& r, int k, uint32_t* own) {
  const int i = threadIdx.x;
  const uint32_t mine = *own = i >= GROUPS ? 0 : r.blocks > 1 ? peer32(&r.s.crest[i % r.crests], i / r.crests) : r.s.crest[i];
  uint32_t low = 0;
#pragma unroll 1
  for (uint32_t bit = 1u << 31; bit >= 1u << 10; bit >>= 1)
    if (__syncthreads_count(mine >= (low | bit)) >= k) low |= bit;
  return low > KEY_NONE ? of_key(low) : LEAST;
}

// Sum over the cluster of every thread's v; slot: a word of each block's that nothing else has used since the last two meetings.
template <int THREADS>
__device__ __forceinline__ uint64_t cluster_sum(const Row& r, uint64_t v, uint64_t* slot) {
  v = block_sum64<THREADS>(v, r.s.red);
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
template <int THREADS>
__device__ __forceinline__ void end_row(const Row& r, const DrawArgs& a, int64_t row, int keep, uint64_t want, bool p_of_kept, float top_p, uint64_t least, float u) {
  Shared& s = r.s;
  const int n = min((int)s.n_list, keep), i = threadIdx.x;
  const uint64_t p = i < n ? s.list.by_rank[i] : 0;
  uint64_t w = i < n ? r.weight(of_place(p)) : 0, all;
  const uint64_t before = block_before64<THREADS>(w, s.red, &all);
  if (p_of_kept) {  // top_p of what top_k kept
    bool lost;
    want = share_of(all, top_p, &lost);
    want += lost;
    if (want < 1) want = 1;
  }
  if (want && before >= want) w = 0;
  if (w < least) w = 0;
  __syncthreads();
  // in the order of the indices, which falling (2^20 - 1 - index, weight) is: 20 bits and 44
  const int kept = __syncthreads_count(w != 0);
  const uint64_t total = block_sum64<THREADS>(w, s.red2);
  bool lost;
  const uint64_t target = share_of(total, u, &lost);
  const uint64_t member = sorted<THREADS>(w ? (p & 0xFFFFF) << 44 | w : 0, kept, s.list.place);  // the kept ones are a beginning of the order
  const uint64_t mine = member & ((1ull << 44) - 1), front = block_before64<THREADS>(mine, s.red, &all);
  if (front <= target && front + mine > target) {  // one thread
    a.out[row] = 0xFFFFF - (int)(member >> 44);
    if (a.prob) a.prob[row] = (float)((double)mine / (double)total);
  }
}

// The row of this block, one to a block and at most a row per thread: first those whose top_p has no short list behind top_k, which take two to four times as
// long as others (256 rows of mixed wishes: 219 us in the order of the rows, 171 so; 2 us where all are alike).
template <int THREADS>
__device__ __forceinline__ int long_ones_first(Shared& s, const DrawArgs& a) {
  const int m = threadIdx.x, warp = m >> 5, lane = m & 31;
  bool is_long = false;
  if (m < a.M) {
    is_long = a.top_p && a.top_p[m] < 1.f && !sb_draw_lists(a.top_k ? sb_draw_top_k(a.top_k[m], a.N) : 0) && (!a.temperature || a.temperature[m] > 0.f);
  }
  const unsigned who = __ballot_sync(0xffffffffu, is_long);
  if (lane == 0) s.red[warp] = __popc(who);
  const int all = __syncthreads_count(is_long);
  int before = 0;
  for (int i = 0; i < warp; i++) before += (int)s.red[i];
  before += __popc(who & ((1u << lane) - 1));  // long ones in front of row m
  if (m < a.M && (is_long ? before : all + m - before) == (int)blockIdx.x) s.there = m;
  __syncthreads();
  const int row = (int)s.there;
  __syncthreads();
  return row;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) draw_kernel(const __grid_constant__ DrawArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *(Shared*)smem;
  float* queue = (float*)(smem + (sizeof(Shared) + 15) / 16 * 16);  // 64 logits of each warp
  float* near = queue + THREADS * 2;
  pdl_wait();
  pdl_trigger();
  uint32_t rank, blocks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
  const int64_t row = THREADS == 1024 && blocks == 1 && a.M <= THREADS ? long_ones_first<THREADS>(s, a) : blockIdx.x / blocks;
  const int span = ((a.N + (int)blocks - 1) / (int)blocks + 7) / 8 * 8;
  Row r{s, near};
  r.x = (const char*)a.x + row * a.ld * (a.f32 ? 4 : 2);
  r.f32 = a.f32;
  r.blocks = (int)blocks;
  r.rank = (int)rank;
  r.first = min(a.N, (int)rank * span);
  r.share = min(a.N - r.first, span);
  r.held = min(r.share, share_kept<THREADS>()) & ~3;
  r.vec = ((uintptr_t)r.x & 15) == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  float top = -INFINITY;
  int top_q = -1;  // a thread's indices rise, and NaN is not larger
  constexpr int AHEAD = 5;
#pragma unroll 1
  for (int q0 = threadIdx.x; q0 < (r.share + 3) / 4; q0 += THREADS * AHEAD) {
    float4 v[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; e++) v[e] = r.far(q0 + e * THREADS);
#pragma unroll
    for (int e = 0; e < AHEAD; e++) {
      const int q = q0 + e * THREADS;
      if (q < r.held / 4) ((float4*)near)[q] = v[e];
      const float l = fmaxf(fmaxf(v[e].x, v[e].y), fmaxf(v[e].z, v[e].w));
      if (l > top) top = l, top_q = q;
    }
  }
  int top_at = 0;
  if (top_q >= 0) {
    const float4 v = r.quad(top_q);  // what this thread has written
    top_at = top_q * 4 + (v.x == top ? 0 : v.y == top ? 1 : v.z == top ? 2 : 3);
  }
  uint64_t best = top > -INFINITY ? r.place(top, top_at) : 0;
  // groups of neighbouring threads
  r.crests = GROUPS / r.blocks;
  const int group = THREADS / r.crests;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (o == group && lane % o == 0) s.crest[threadIdx.x / o] = (uint32_t)(best >> 20);
    const uint64_t v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if (threadIdx.x < 512) s.fraction[threadIdx.x] = __double_as_longlong(exp2(43.0 + threadIdx.x / 8 / 64.0));
  if (threadIdx.x == 0) s.n_list = 0;
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  for (int i = 0; i < (THREADS / 32); i++) best = s.red[i] > best ? s.red[i] : best;
  const float heat = a.temperature ? a.temperature[row] : 1.f;  // read by all blocks before one of them may write a result
  if (threadIdx.x == 0) s.best = best;
  r.meet();
  if (r.blocks > 1) {
    uint64_t v[MAX_CLUSTER];
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++) v[b] = b < r.blocks ? peer64(&s.best, b) : 0;
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++) best = v[b] > best ? v[b] : best;
  }
  const bool none = best >> 20 <= KEY_NONE;
  if (none || !(heat > 0.f)) {
    if (rank == 0 && threadIdx.x == 0) {
      a.out[row] = none ? -1 : 0xFFFFF - (int)(best & 0xFFFFF);
      if (a.prob) a.prob[row] = none ? 0.f : 1.f;
    }
    r.meet();
    return;
  }
  r.m32 = of_place(best);
  r.m = (double)fminf(r.m32, -LEAST);
  // beside +inf nothing has a weight
  r.scale = r.m32 == INFINITY ? 1e30 : 64 * 1.4426950408889634074 / heat;
  // 45 * 64 further down; to the next float above, since of the logits only floats are asked about
  r.least_l = r.m32 == INFINITY ? INFINITY : r.scale > 0 ? __double2float_ru(r.m - 2880.0 / r.scale) : LEAST;
  r.zero_l = __double2float_rd(r.m - 2944.0 / r.scale);
  const double down = (r.m - (double)r.zero_l) * r.scale;  // what is left of it where floats lie far apart
  r.plain = r.m32 < INFINITY && r.scale > 0 && r.zero_l >= LEAST && down >= 2912.0 && down <= 60000.0;
  r.bin_scale = fmaxf(1e-36f, fminf((BINS - 1) / (32.f * heat), 1e30f));  // never 0: infinities are far from or in front of numbers at any heat
  if (r.m32 == INFINITY) r.m32 = -LEAST;  // bins below a largest logit of +inf: that one in the first, whatever is finite by its distance from the largest number
  const int k = a.top_k ? sb_draw_top_k(a.top_k[row], a.N) : 0;
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
    float low = of_place(from);
    if (!sums) {
      if (k == 0) continue;
      if (sb_draw_lists(k)) {
        uint32_t own;
        gather<THREADS>(r, crest_bound<THREADS>(r, k, &own), INFINITY, [](float, uint64_t) { return true; });
        few = (r.blocks > 1 ? peer32(&s.n_list, 0) : s.n_list) <= LIST;
        if (few) {
          if (r.rank == 0) rank_list<THREADS>(s, (int)s.n_list);
          break;
        }
        r.meet();  // the number has been read
      }
      uint64_t there = 0;
      each<THREADS>(r, LEAST, [&](float, int, bool in) { there += in; });
      if ((uint64_t)k >= cluster_sum<THREADS>(r, there, &s.there)) continue;  // all that have any weight are kept
      want = k;
    } else {
      if (!(top_p < 1.f)) continue;
      uint64_t sum = 0;
      const bool by_key = (from & 0xFFFFF) == 0;
      if (by_key && r.plain) {
        const float cut = fmaxf(low, r.least_l);
        const int near = r.held / 4, all = (r.share + 3) / 4;
#pragma unroll 1
        for (int q = threadIdx.x; q < near; q += THREADS) sum += r.weights(((const float4*)r.near)[q], cut);
#pragma unroll 1
        for (int q = near + threadIdx.x; q < all; q += 2 * THREADS) {
          const float4 v0 = r.far(q), v1 = r.far(q + THREADS);
          sum += r.weights(v0, cut) + r.weights(v1, cut);
        }
      } else {
        each<THREADS>(r, low, [&](float l, int i, bool in) {
          const uint64_t w = r.weight(l);
          sum += in && (by_key || r.place(l, i) >= from) ? w : 0;
        });
      }
      sum = cluster_sum<THREADS>(r, sum, &s.weights);
      bool lost;
      want = share_of(sum, top_p, &lost);
      want = max((uint64_t)1, want + lost);
      // The 256 largest and some more usually hold top_p. They hold little more than the largest of the groups: where those do not come near,
      // the pass is saved.
      bool near_it = false;
      float bound = 0.f;
      if (!sb_draw_lists(k)) {
        uint32_t own;
        bound = fmaxf(low, crest_bound<THREADS>(r, GROUPS / 2, &own));
        const uint64_t crests = block_sum64<THREADS>(of_key(own) >= bound ? r.weight(of_key(own)) : 0, s.red);
        near_it = crests + crests / 16 >= want;
      }
      if (near_it) {
        if (r.rank == 0 && threadIdx.x == 0) s.n_list = 0;
        r.meet();
        gather<THREADS>(r, bound, INFINITY, [&](float, uint64_t p) { return p >= from; });
        if (r.rank == 0) {
          const int n = (int)s.n_list;
          uint64_t w = 0;
          if (n <= LIST) w = block_sum64<THREADS>(threadIdx.x < n ? r.weight(of_place(s.list.place[threadIdx.x])) : 0, s.red);
          if (threadIdx.x == 0) s.word = w >= want;
        }
        r.meet();
        few = peer64(&s.word, 0);
        if (few) {
          if (r.rank == 0) rank_list<THREADS>(s, (int)s.n_list);
          break;
        }
        r.meet();  // the word has been read
      }
      // logits that far down stay out of the bins: the cut is above them
      const float reach = sb_draw_reach(sum, want, a.N, heat, r.m32);
      if (reach < 1e30f) low = fmaxf(low, r.m32 - reach);
      // bins of what is left
      const float width = r.m32 - low;
      if (width < 32.f * heat) r.bin_scale = fminf((BINS - 1) / width, 1e30f);
    }
    int b0 = 0, hi = 52;
    uint64_t known = 0, left = want;
    bool digits = false;  // within bin b0, where more than LIST share it: by the next ten bits of the place
#pragma unroll 1
    while (true) {
      const int lo = max(0, hi - 10), mask = (1 << (hi - lo)) - 1;
      clear_bins<THREADS>(s, sums);
      if (digits) {
        each<THREADS>(r, low, [&](float l, int i, bool in) {
          const uint64_t p = r.place(l, i);
          in = in && p >= from && r.bin(l) == b0 && (hi == 52 || p >> hi == known);
          if (in) add_to_bin(s, sums, mask - ((int)(p >> lo) & mask), sums ? r.weight(l) : 0);  // larger digits first
        });
      } else {
        // Often few logits go into bins, but some of nearly every warp's: they queue, and 32 at a time are weighed and added.
        float* line = queue + warp * 64;
        int n = 0;
        auto weigh = [&](float l) { add_to_bin(s, sums, r.bin(l), sums ? r.weight(l) : 0); };
        const bool by_key = (from & 0xFFFFF) == 0;  // `from` begins a key
        const int all = (r.share + 3) / 4;
        auto get = [&](int q) { return q < all ? r.quad(q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); };
        float4 ahead[3];  // requested before they are needed: far ones come from memory
#pragma unroll
        for (int e = 0; e < 3; e++) ahead[e] = get(warp * 32 + lane + e * THREADS);
#pragma unroll 1
        for (int q0 = warp * 32; q0 < all; q0 += THREADS) {
          const int q = q0 + lane;
          const float4 v = ahead[0];
          ahead[0] = ahead[1];
          ahead[1] = ahead[2];
          ahead[2] = get(q + 3 * THREADS);
          if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= low)) continue;
          const float one[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const bool in = one[e] >= low && (by_key || r.place(one[e], q * 4 + e) >= from);
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (in) line[n + __popc(who & ((1u << lane) - 1))] = one[e];
            n += __popc(who);
            if (n >= 32) {
              __syncwarp();
              const float l = line[lane], next = line[32 + lane];
              __syncwarp();
              line[lane] = next;
              n -= 32;
              weigh(l);
            }
          }
        }
        __syncwarp();
        if (lane < n) weigh(line[lane]);
      }
      const Crossing c = cross<THREADS>(r, sums, left);
      if (c.count == 0) break;  // not reached: the bins hold `left`. Without it there is no cut.
      left = c.want;
      if (digits) {
        known = (hi < 52 ? known << (hi - lo) : 0) | (uint64_t)(mask - c.bin);
        hi = lo;
      } else {
        b0 = c.bin;
        few = c.front + c.count <= LIST;
      }
      if (few || c.count <= LIST) {
        // logits of bin b0 and in front of it, and a little more: the bin itself is looked at in what is left
        const float slack = fabsf(r.m32) * 1e-6f, deep = (b0 + 1.01f) / r.bin_scale + slack, flat = (b0 - 0.01f) / r.bin_scale - slack;
        gather<THREADS>(r, b0 < BINS - 1 && deep < 1e30f ? fmaxf(low, r.m32 - deep) : low, !few && flat > 0.f && flat < 1e30f ? r.m32 - flat : INFINITY, [&](float l, uint64_t p) {
          const int b = r.bin(l);
          return p >= from && (few ? b <= b0 : b == b0 && (!digits || p >> hi == known));
        });
        if (r.rank == 0) {
          const int n = (int)s.n_list;
          rank_list<THREADS>(s, n);
          if (!few && !sums && threadIdx.x == 0) s.word = s.list.by_rank[left - 1];
          if (!few && sums) {
            uint64_t all;
            const uint64_t w = threadIdx.x < n ? r.weight(of_place(s.list.by_rank[threadIdx.x])) : 0, before = block_before64<THREADS>(w, s.red, &all);
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
      end_row<THREADS>(r, a, row, by_count ? k : LIST, by_count ? 0 : want, by_count && top_p < 1.f, top_p, least, u);
    }
    r.meet();
    return;
  }
  // The draw: a warp sums pieces of 512 keys, the sums in front of the pieces tell which holds the token, and one warp looks through that piece.
  const float low = of_place(from);
  const bool by_key = (from & 0xFFFFF) == 0;
  auto kept = [&](float l, int i) -> uint64_t {
    const uint64_t w = r.weight(l);
    return l >= low && (by_key || r.place(l, i) >= from) && w >= least ? w : 0;
  };
  const bool simple = by_key && r.plain && least <= 1;
  const float cut = fmaxf(low, r.least_l);
  auto kept4 = [&](const float4& v, int q) -> uint64_t {
    if (simple) return r.weights(v, cut);
    if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= low)) return 0;
    return kept(v.x, q * 4) + kept(v.y, q * 4 + 1) + kept(v.z, q * 4 + 2) + kept(v.w, q * 4 + 3);
  };
  const int pieces = (r.share + 4 * PIECE - 1) / (4 * PIECE);
  uint64_t* piece_sum = s.piece_sum;  // bins and list are done with
#pragma unroll 1
  for (int p = warp; p < pieces; p += THREADS / 32) {
    float4 v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = r.quad(p * PIECE + e * 32 + lane);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) sum += kept4(v[e], p * PIECE + e * 32 + lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) piece_sum[p] = sum;
  }
  __syncthreads();
  const int each_thread = (pieces + THREADS - 1) / THREADS, p0 = threadIdx.x * each_thread;
  uint64_t mine = 0, block_total, total = 0;
  for (int p = p0; p < min(pieces, p0 + each_thread); p++) mine += piece_sum[p];
  uint64_t before = block_before64<THREADS>(mine, s.red, &block_total);
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
  const unsigned owner = __ballot_sync(0xffffffffu, target >= before && target < before + mine);
  if (!owner) return;
  const int src = __ffs(owner) - 1;
  before = __shfl_sync(0xffffffffu, before, src);
  int p = __shfl_sync(0xffffffffu, p0, src);
  while (before + piece_sum[p] <= target) before += piece_sum[p++];
#pragma unroll 1
  for (int q = p * PIECE + lane; ; q += 32) {
    const float4 v = r.quad(q);
    const uint64_t w = kept4(v, q);
    uint64_t sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + sum > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        uint64_t up_to = before + sum - w;
        const float one[4] = {v.x, v.y, v.z, v.w};
        bool found = false;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint64_t we = kept(one[e], q * 4 + e);
          up_to += we;
          if (!found && up_to > target) {
            found = true;
            a.out[row] = r.first + q * 4 + e;
            if (a.prob) a.prob[row] = (float)((double)we / (double)total);
          }
        }
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
    if (q - lane >= pieces * PIECE) return;  // not reached: the sums say that it is here
  }
}

}  // namespace

int k_draw(strictb200_ctx* ctx, const void* x, int f32, int64_t M, int64_t N, int64_t ld, const float* u, const float* temperature, const int32_t* top_k,
           const float* top_p, const float* min_p, int32_t* out, float* prob) {
  // Blocks look at other rows' wishes for their order, unless those are written over by the results.
  auto over = [&](const void* result, const void* wish) {
    const uintptr_t r = (uintptr_t)result, w = (uintptr_t)wish, bytes = (uintptr_t)M * 4;
    return result && wish && r < w + bytes && w < r + bytes;
  };
  bool in_order = false;
  for (const void* wish : {(const void*)temperature, (const void*)top_k, (const void*)top_p}) in_order |= over(out, wish) || over(prob, wish);
  const DrawArgs a{x, ld, (int)N, f32, in_order ? INT32_MAX : (int)M, u, temperature, top_p, min_p, top_k, out, prob};
  // Few rows: eight blocks of 512 threads for a long one, fewer where they hold it. Many rows: blocks of 1024 threads that have an SM each, as few to a row as keeps the SMs busy.
  int blocks = 1;
  while (blocks < MAX_CLUSTER && N > (int64_t)blocks * share_kept<512>()) blocks *= 2;
  const bool many = M * blocks > ctx->sm_count && blocks > 1;
  if (many)
    while (blocks > 1 && M * blocks > (blocks > 2 ? ctx->sm_count * 7 / 8 : ctx->sm_count)) blocks /= 2;  // clusters of four do not fill every SM
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16;
  const size_t smem = fixed + (many ? 1024 : 512) * 8 + (size_t)std::min<int64_t>(many ? share_kept<1024>() : share_kept<512>(), (N + blocks - 1) / blocks + 8) * 4;
  const auto kernel = many ? draw_kernel<1024> : draw_kernel<512>;
  static SbDeviceOnce once;
  SB_CUDA(once.run(ctx->device, [&] {
    const cudaError_t e = cudaFuncSetAttribute(draw_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fixed + 512 * 8 + share_kept<512>() * 4);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(draw_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fixed + 1024 * 8 + share_kept<1024>() * 4);
  }));
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
    SB_CUDA(sb_launch_cluster(ctx, kernel, dim3((unsigned)(std::min(M - m0, most) * blocks)), dim3(many ? 1024 : 512), smem, dim3((unsigned)blocks), part));
    ctx->launches++;
  }
  return STRICTB200_OK;
}
