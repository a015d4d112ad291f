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
//   top_k of up to 128: the k-th largest of those groups' places bounds the first k tokens from below, and what lies above it, seldom more than
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
  l = l != l ? -INFINITY : l + 0.f;
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
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
  // what blocks tell one another: largest place and number of a share that has any weight, a cut, the kept weights
  uint64_t best, there, word, drawn;
  uint32_t n_list;
  long long fraction[64];  // bits of 2^(43 + i / 64)
  uint64_t crest[THREADS], crest_own[THREADS];  // largest places of groups of threads: of all blocks, of this one
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
  double m, scale;     // its value, 64 log2(e) / temperature
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
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    if (k == top) return 1ull << 43;
    if (k <= KEY_NONE || top >= KEY_INF) return 0;  // beside +inf nothing has a weight
    // the float's bits as a double's (a subnormal one becomes another of no consequence)
    const uint32_t b = __float_as_uint(of_key(k));
    const double d = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(b << 29)) - m;
    constexpr double WHOLE = 6755399441055744.0;  // 1.5 * 2^52
    if (!(d * scale > -2880.0)) return 0;  // 2^-45
    const double t = fma(d, scale, WHOLE), f = fma(d, scale, WHOLE - t);
    const int n = __double2loint(t);
    constexpr double C = 0.69314718055994530942 / 64;
    double p = C * C * C * C / 24;
    p = fma(p, f, C * C * C / 6);
    p = fma(p, f, C * C / 2);
    p = fma(p, f, C);
    p = fma(p, f, 1.0);
    const long long two = s.fraction[n & 63] + ((long long)(n >> 6) << 52);  // 2^(43 + n / 64)
    return (uint64_t)__double_as_longlong(fma(p, __longlong_as_double(two), 4503599627370496.0)) - 0x4330000000000000ull;
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
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < WARPS; i++) s += red[i];
  return s;
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
  uint64_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; i++) {
    if (i < warp) before += red[i];
    total += red[i];
  }
  *all = total;
  return before + sum - v;
}

// The bin where a running sum over the bins (SUMS: of weights, otherwise of counts) reaches `want`; want == 0 and share_p >= 0: share_p of all the weights.
struct Crossing {
  int bin;
  uint64_t count;         // members of the bin
  uint64_t front;         // members of the bins in front
  uint64_t want;          // of the bin's own
  bool whole;             // the bin is kept as a whole
};
template <bool SUMS>
__device__ Crossing cross(Row& r, uint64_t* want, float share_p) {
  Shared& s = r.s;
  const int per = BINS / r.blocks;
  r.meet();  // all bins are counted
  const uint32_t* counts = s.bin.count;
  auto sum_of = [&](int i) { return s.bin.sum[0][i] + ((uint64_t)s.bin.sum[1][i] << 15) + ((uint64_t)s.bin.sum[2][i] << 30); };
  int owner = 0;
  uint64_t front_c = 0, front_s = 0, all_s = 0;
  if (r.blocks > 1) {
    uint64_t tc = 0, ts = 0;
    for (int i = threadIdx.x; i < per; i += THREADS) {
      uint32_t c[MAX_CLUSTER];
      uint64_t w[MAX_CLUSTER];
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++)
        if (b < r.blocks) {
          c[b] = peer32(&s.bin.count[r.rank * per + i], b);
          if (SUMS) {
            const int at = r.rank * per + i;
            w[b] = peer32(&s.bin.sum[0][at], b) + ((uint64_t)peer32(&s.bin.sum[1][at], b) << 15) + ((uint64_t)peer32(&s.bin.sum[2][at], b) << 30);
          }
        }
      uint64_t cc = 0, ww = 0;
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++)
        if (b < r.blocks) {
          cc += c[b];
          if (SUMS) ww += w[b];
        }
      s.part_count[i] = (uint32_t)cc;
      if (SUMS) s.part_sum[i] = ww;
      tc += cc;
      ts += ww;
    }
    tc = block_sum64(tc, s.red);
    if (SUMS) ts = block_sum64(ts, s.red2);
    if (threadIdx.x == 0) s.total_count = tc, s.total_sum = ts;
    r.meet();
    uint64_t c[MAX_CLUSTER], w[MAX_CLUSTER];
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++)
      if (b < r.blocks) {
        c[b] = peer64(&s.total_count, b);
        w[b] = SUMS ? peer64(&s.total_sum, b) : 0;
        all_s += w[b];
      }
    if (SUMS && share_p >= 0.f) {
      bool lost;
      *want = share_of(all_s, share_p, &lost);
      *want += lost;
      if (*want < 1) *want = 1;
    }
    owner = r.blocks - 1;
    bool found = false;
#pragma unroll
    for (int b = 0; b < MAX_CLUSTER; b++)
      if (b < r.blocks && !found) {
        if ((SUMS ? front_s + w[b] : front_c + c[b]) >= *want) owner = b, found = true;
        else front_c += c[b], front_s += w[b];
      }
  } else if (SUMS && share_p >= 0.f) {
    uint64_t ts = 0;
    for (int i = threadIdx.x; i < per; i += THREADS) ts += sum_of(i);
    all_s = block_sum64(ts, s.red2);
    bool lost;
    *want = share_of(all_s, share_p, &lost);
    *want += lost;
    if (*want < 1) *want = 1;
  }
  // the owner's part, two neighbouring bins per thread at most
  uint64_t c2[2] = {0, 0}, w2[2] = {0, 0};
  const int each = (per + THREADS - 1) / THREADS;
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int i = threadIdx.x * each + e;
    if (e < each && i < per) {
      c2[e] = r.blocks > 1 ? peer32(&s.part_count[i], owner) : counts[i];
      if (SUMS) w2[e] = r.blocks > 1 ? peer64(&s.part_sum[i], owner) : sum_of(i);
    }
  }
  uint64_t all, before_c = front_c + block_before64(c2[0] + c2[1], s.red, &all), before_s = 0;
  if (SUMS) before_s = front_s + block_before64(w2[0] + w2[1], s.red2, &all);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const uint64_t here = SUMS ? w2[e] : c2[e], before = SUMS ? before_s : before_c;
    if (e < each && before < *want && before + here >= *want) {  // one thread, once
      s.pick[0] = owner * per + threadIdx.x * each + e;
      s.pick[1] = c2[e];
      s.pick[2] = before_c;
      s.pick[3] = *want - before;
      s.pick[4] = SUMS ? c2[e] == 1 : here == *want - before;
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

// A member into its bin. Where a warp's members all go to one bin (rows of equal logits, large temperatures) they go together.
template <bool SUMS>
__device__ __forceinline__ void add_to_bin(Shared& s, bool in, int b, uint64_t w) {
  const unsigned who = __ballot_sync(0xffffffffu, in);
  if (!who) return;
  const int lead = __ffs(who) - 1, b0 = __shfl_sync(0xffffffffu, b, lead);
  uint32_t n = 1;
  if (__all_sync(0xffffffffu, !in || b == b0)) {
    if (SUMS) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    }
    n = __popc(who);
    in = (threadIdx.x & 31) == lead;
  }
  if (!in) return;
  atomicAdd(&s.bin.count[b], n);
  if (SUMS && w) {  // at most 2^48
    atomicAdd(&s.bin.sum[0][b], (uint32_t)w & 0x7FFFu);
    atomicAdd(&s.bin.sum[1][b], (uint32_t)(w >> 15) & 0x7FFFu);
    atomicAdd(&s.bin.sum[2][b], (uint32_t)(w >> 30));
  }
}

// The members `of` chooses, from all blocks, into the first block's list (at most LIST of them).
// AGAIN: the place of the list was in use.
template <bool AGAIN, typename F>
__device__ void gather(Row& r, F&& of) {
  Shared& s = r.s;
  if (AGAIN) {
    r.meet();  // nobody reads bins any more
    if (r.rank == 0 && threadIdx.x == 0) s.n_list = 0;
    r.meet();
  }
  for (int i = threadIdx.x; i < r.share; i += THREADS) {
    const uint32_t k = r.key(i);
    const uint64_t p = r.place(k, i);
    if (!of(k, p)) continue;
    uint32_t at;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(remote(&s.n_list, 0)) : "memory");
    if (at < LIST) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&s.list.place[at], 0)), "l"(p) : "memory");
  }
  r.meet();
}

// Ranks of the list's members (the first block): by_rank. Threads share out the comparisons.
__device__ void rank_list(Shared& s, int n) {
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

// Lowest place that is kept when the order is cut, among the places from `from` on: after `want` tokens, or (SUMS) where the weight in front reaches share_p of theirs.
// *few: at most LIST places are kept, and the first block has them and the rest of their bin in its list, ranked; then the value is the cut for COUNTS and not
// yet known for SUMS (*want: the weight to be reached).
template <bool SUMS>
__device__ uint64_t cut(Row& r, uint64_t from, uint64_t* want, float share_p, bool* few) {
  Shared& s = r.s;
  clear_bins(s, SUMS);
  for (int i0 = 0; i0 < r.share; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < r.share ? r.key(i) : 0;
    const bool in = i < r.share && r.place(k, i) >= from;
    add_to_bin<SUMS>(s, in, in ? r.bin(k) : 0, SUMS && in ? r.weight(k) : 0);
  }
  Crossing c = cross<SUMS>(r, want, share_p);
  const int b0 = c.bin;
  *few = c.front + c.count <= LIST;
  if (*few) {
    gather<true>(r, [&](uint32_t k, uint64_t p) { return p >= from && r.bin(k) <= b0; });
    if (r.rank == 0) rank_list(s, (int)s.n_list);
    return 0;
  }
  uint64_t known = 0, low_place = 0;
  int shift = 52;
  bool done = false;
  while (!done) {
    if (c.whole && shift < 52) {  // of the bins of a digit: all that begin with it
      low_place = known << shift;
      break;
    }
    if (c.count <= LIST) {
      const int sh = shift;
      const uint64_t kn = known;
      gather<true>(r, [&](uint32_t k, uint64_t p) { return p >= from && r.bin(k) == b0 && (sh == 52 || p >> sh == kn); });
      if (r.rank == 0) {
        const int n = (int)s.n_list;
        rank_list(s, n);
        if (!SUMS) {
          if (threadIdx.x == 0) s.word = s.list.by_rank[c.want - 1];
        } else {
          for (int i = threadIdx.x; i < n; i += THREADS) s.list.w[i] = r.weight((uint32_t)(s.list.by_rank[i] >> 20));
          __syncthreads();
          uint64_t all;
          const uint64_t w = threadIdx.x < n ? s.list.w[threadIdx.x] : 0, before = block_before64(w, s.red, &all);
          if (before < c.want && before + w >= c.want) s.word = s.list.by_rank[threadIdx.x];
        }
      }
      r.meet();
      low_place = peer64(&s.word, 0);
      r.meet();
      break;
    }
    // more than LIST in one bin: by the next ten bits of the place
    const int low = max(0, shift - 10), bits = shift - low;
    r.meet();
    clear_bins(s, SUMS);
    for (int i0 = 0; i0 < r.share; i0 += THREADS) {
      const int i = i0 + threadIdx.x;
      const uint32_t k = i < r.share ? r.key(i) : 0;
      const uint64_t p = r.place(k, i);
      const bool in = i < r.share && p >= from && r.bin(k) == b0 && (shift == 52 || p >> shift == known);
      const int d = (1 << bits) - 1 - ((int)(p >> low) & ((1 << bits) - 1));  // larger digits first
      add_to_bin<SUMS>(s, in, in ? d : 0, SUMS && in ? r.weight(k) : 0);
    }
    uint64_t inner = c.want;
    c = cross<SUMS>(r, &inner, -1.f);
    known = (shift < 52 ? known << bits : 0) | (uint64_t)((1 << bits) - 1 - c.bin);
    shift = low;
  }
  return low_place > from ? low_place : from;
}

// The row's end in the first block, from its ranked list: `keep` of it are the kept beginning, or, with want > 0, those up to the weight `want`.
__device__ void end_row(Row& r, const DrawArgs& a, int64_t row, int keep, uint64_t want, bool p_of_kept, float top_p, uint64_t least, float u) {
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

  uint64_t best = 0, there = 0;  // the first of the order; how many are not -inf
  auto take = [&](uint32_t k, int i) {
    if (i < r.held) keys[i] = k;
    there += k > KEY_NONE;
    const uint64_t p = r.place(k, i);
    best = p > best ? p : best;
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
          take(key_of(v[e].x), i);
          take(key_of(v[e].y), i + 1);
          take(key_of(v[e].z), i + 2);
          take(key_of(v[e].w), i + 3);
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
  // 512 groups in the cluster: threads of a block, or two, four or eight neighbours
  r.crests = THREADS / r.blocks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (o == r.blocks && lane % o == 0) s.crest_own[threadIdx.x / o] = best;
    const uint64_t v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if (threadIdx.x < 64) s.fraction[threadIdx.x] = __double_as_longlong(exp2(43.0 + threadIdx.x / 64.0));
  if (threadIdx.x == 0) s.n_list = 0;
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  for (int i = 0; i < WARPS; i++) best = s.red[i] > best ? s.red[i] : best;
  there = block_sum64(there, s.red2);
  if (threadIdx.x == 0) s.best = best, s.there = there;
  r.meet();
  if (r.blocks > 1) {
    there = 0;
    for (int b = 0; b < r.blocks; b++) {
      const uint64_t v = peer64(&s.best, b);
      best = v > best ? v : best;
      there += peer64(&s.there, b);
    }
  }
  r.top = (uint32_t)(best >> 20);
  r.m32 = of_key(r.top);
  r.m = r.m32;
  const float heat = a.temperature ? a.temperature[row] : 1.f;
  if (r.top <= KEY_NONE || !(heat > 0.f)) {
    if (rank == 0 && threadIdx.x == 0) {
      a.out[row] = r.top <= KEY_NONE ? -1 : 0xFFFFF - (int)(best & 0xFFFFF);
      if (a.prob) a.prob[row] = r.top <= KEY_NONE ? 0.f : 1.f;
    }
    r.meet();
    return;
  }
  r.scale = 64 * 1.4426950408889634074 / heat;
  r.bin_scale = fminf((BINS - 1) / (32.f * heat), 1e30f);
  if (r.top >= KEY_INF) r.m32 = 3.4028235e38f;  // bins below a largest logit of +inf: that one in the first, whatever is finite by its distance from the largest number
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
  const uint64_t least = min_p > 0.f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * ONE) : 0;
  float u = a.u[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  uint64_t from = (uint64_t)(KEY_NONE + 1) << 20, want = 0;
  bool few = false;
  if (k > 0 && k < a.N && 4 * k <= r.blocks * r.crests) {
    // The k-th largest of the groups' largest places has at least k places from it on, and, where the largest are not all in a few groups, not many more.
    uint64_t* crest = s.crest;
    const int n = r.blocks * r.crests;
    uint64_t mine = 0;
    if (threadIdx.x < n) mine = r.blocks > 1 ? peer64(&s.crest_own[threadIdx.x % r.crests], threadIdx.x / r.crests) : s.crest_own[threadIdx.x];
    crest[threadIdx.x] = mine;
    if (threadIdx.x == 0) s.pick[0] = 0;  // fewer than k groups have any
    __syncthreads();
    if (threadIdx.x < n) {
      int above = 0;
      for (int j = 0; j < n; j++) above += crest[j] > mine;
      if (above == k - 1) s.pick[0] = mine;
    }
    __syncthreads();
    const uint64_t low = s.pick[0] > from ? s.pick[0] : from;
    gather<false>(r, [&](uint32_t, uint64_t p) { return p >= low; });
    few = (r.blocks > 1 ? peer32(&s.n_list, 0) : s.n_list) <= LIST;
    if (few && r.rank == 0) {
      rank_list(s, (int)s.n_list);
      end_row(r, a, row, k, 0, top_p < 1.f, top_p, least, u);
    }
    if (!few) r.meet();  // the number has been read
  }
  if (!few && k > 0 && k < a.N) {
    want = k;
    if (want < there) {  // otherwise all that have any weight are kept
      from = cut<false>(r, from, &want, -1.f, &few);
      if (few && r.rank == 0) end_row(r, a, row, k, 0, top_p < 1.f, top_p, least, u);
    }
  }
  if (!few && top_p < 1.f) {
    from = cut<true>(r, from, &want, fmaxf(top_p, 0.f), &few);
    if (few && r.rank == 0) end_row(r, a, row, LIST, want, false, top_p, least, u);
  }
  if (few) {
    r.meet();
    return;
  }
  // The draw: a thread sums a contiguous part of the block's share (an odd number of keys, so that a warp's reads meet no bank twice), the sums in front of
  // it tell the one thread whose part holds the token, and its warp looks through that part.
  const int each_thread = (r.share + THREADS - 1) / THREADS | 1, i0 = min(r.share, (int)threadIdx.x * each_thread), i1 = min(r.share, i0 + each_thread);
  auto kept = [&](int i) -> uint64_t {
    const uint32_t key = r.key(i);
    if (r.place(key, i) < from) return 0;
    const uint64_t w = r.weight(key);
    return w >= least ? w : 0;
  };
  uint64_t mine = 0, block_total, total = 0;
#pragma unroll 4
  for (int i = i0; i < i1; i++) mine += kept(i);
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
