// Norm and rotation of the new tokens' heads, keys and values into the pages of a cache.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace {

struct Rates {
  double turn[64];  // theta^(-2i/D) / (2 pi): turns per position of the pair i
};

struct Eight {
  float2 v[4];
};
__device__ __forceinline__ Eight unpacked(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  Eight r;
#pragma unroll
  for (int e = 0; e < 4; e++) r.v[e] = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u));
  return r;
}
__device__ __forceinline__ uint4 packed(const Eight& r) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const __nv_bfloat162 y = __float22bfloat162_rn(r.v[e]);
    w[e] = *(const uint32_t*)&y;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ Eight eight(const float* p, int further) {
  const float4 a = *(const float4*)p, b = *(const float4*)(p + further);
  return Eight{{{a.x, a.y}, {a.z, a.w}, {b.x, b.y}, {b.z, b.w}}};
}

// Sequence of packed row t (0 <= t < T), the first b with t < starts[b + 1], and the row's position, all of it from one round of loads; B where the row is in
// front of the first or behind the last sequence. All lanes of a warp call it with the same t.
__device__ __forceinline__ int place(const PagedView& v, int64_t t, int* pos) {
  const int lane = threadIdx.x & 31, s0 = v.starts[0];
  for (int b0 = 0; b0 < v.B; b0 += 32) {
    const int b = min(b0 + lane, v.B - 1), end = v.starts[b + 1], back = v.lens[b] - end;
    const unsigned past = __ballot_sync(0xffffffffu, b0 + lane < v.B && t < end);
    if (past) {
      *pos = __shfl_sync(0xffffffffu, back, __ffs(past) - 1) + (int)t;
      return t >= s0 ? b0 + __ffs(past) - 1 : v.B;
    }
  }
  return v.B;
}

// Bound by HBM where there are many tokens: each head is read and written once. A block takes up to 16 neighbouring tokens, whose heads are neighbours in
// memory. All its threads request their share of the first pass over them, then warps look the tokens' places up (a chain of loads, once for all of
// them) and threads make the angles: position times rate in 64 bits, less the whole turns, sine and cosine of the rest in 32. From there on warps go on
// without waiting for one another. D / 16 threads have a head, each eight dims and the eight D / 2 further on, so that a pair meets in one thread.
// (8192 tokens of 48 heads of 128 dims, 201 MB: a token at a time 86 us, places of four tokens looked up at a time 49, this 38;
// 32768 tokens 143 us, 5.6 TB/s; 32 tokens 4.8 us in a graph. Two or three passes requested ahead are 43 to 56 us: fewer blocks fit.)
constexpr int THREADS = 256, MAX_TOKENS = 16;
template <int D>
__global__ void __launch_bounds__(THREADS, 4) rope_paged_kernel(const __grid_constant__ PagedRopeArgs a, const __grid_constant__ Rates r, int tokens) {
  constexpr int LANES = D / 16, PASS = THREADS / LANES;
  __shared__ __align__(16) float cos_s[MAX_TOKENS][D / 2], sin_s[MAX_TOKENS][D / 2];
  __shared__ int64_t row_s[MAX_TOKENS];  // of the token's first key head in the pages; -1: no page, -2: the token belongs to no sequence
  __shared__ int pos_s[MAX_TOKENS];
  const int H = a.Hq + 2 * a.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x % LANES, mine = threadIdx.x / LANES;
  const int pair = threadIdx.x % (D / 2), place_of = pair / 4 % 2 * (D / 4) + pair / 8 * 4 + pair % 4;  // the two fours of a thread apart: no bank conflicts
  const double turn = r.turn[pair];
  pdl_wait();
  pdl_trigger();
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int n = (int)(a.at.T - t0 < tokens ? a.at.T - t0 : tokens), items = n * H;
  const bf16* src = a.qkv + t0 * H * D + 8 * lane;
  struct Share {
    uint4 lo, hi;
  };
  auto request = [&](Share& x, int it) {
    if (it < items) {
      x.lo = *(const uint4*)(src + (int64_t)it * D);
      x.hi = *(const uint4*)(src + (int64_t)it * D + D / 2);
    }
  };
  Share even, odd;
  request(even, mine);
  for (int k = warp; k < n; k += THREADS / 32) {
    int pos = 0;
    const int b = place(a.at, t0 + k, &pos);
    if ((threadIdx.x & 31) == 0) {
      const int page = b < a.at.B && pos >= 0 ? paged_page(a.at, b, pos >> a.at.shift) : -1;
      row_s[k] = b >= a.at.B ? -2 : page < 0 ? -1 : (int64_t)page * a.Hkv * a.at.page + (pos & (a.at.page - 1));
      pos_s[k] = pos;
    }
  }
  __syncthreads();
  for (int k = threadIdx.x / (D / 2); k < n; k += THREADS / (D / 2)) {
    double x = pos_s[k] * turn;
    x -= rint(x);
    sincospif(2.f * (float)x, &sin_s[k][place_of], &cos_s[k][place_of]);
  }
  __syncthreads();
  const float inv_h = 1.0f / H;
  auto process = [&](const Share& x, int it) {
    const bool valid = it < items;  // of all lanes of a head
    const int tok = min((int)((it + 0.5f) * inv_h), n - 1);
    const int h = it - tok * H;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    uint4 y0 = x.lo, y1 = x.hi;
    if (__any_sync(0xffffffffu, valid && !is_v)) {
      Eight x0 = unpacked(y0), x1 = unpacked(y1);
      if (a.qgain) {
        float2 sq = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; e++) sq = __ffma2_rn(x1.v[e], x1.v[e], __ffma2_rn(x0.v[e], x0.v[e], sq));
        float ss = sq.x + sq.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rr = rsqrtf(ss * (1.0f / D) + a.eps);  // 2^-22, far below the rounding to bf16
        const float* gain = (is_q ? a.qgain : a.kgain) + 8 * lane;
        const Eight g0 = eight(gain, 4), g1 = eight(gain + D / 2, 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x0.v[e] = __fmul2_rn(x0.v[e], __fmul2_rn(g0.v[e], make_float2(rr, rr)));
          x1.v[e] = __fmul2_rn(x1.v[e], __fmul2_rn(g1.v[e], make_float2(rr, rr)));
        }
      }
      const Eight c = eight(&cos_s[tok][4 * lane], D / 4), s = eight(&sin_s[tok][4 * lane], D / 4);
      Eight z0, z1;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        z0.v[e] = __ffma2_rn(x0.v[e], c.v[e], __fmul2_rn(x1.v[e], make_float2(-s.v[e].x, -s.v[e].y)));
        z1.v[e] = __ffma2_rn(x1.v[e], c.v[e], __fmul2_rn(x0.v[e], s.v[e]));
      }
      if (!is_v) {
        y0 = packed(z0);
        y1 = packed(z1);
      }
    }
    const int64_t row = row_s[tok];
    if (!valid || row == -2) return;
    bf16* dst;
    if (is_q) {
      dst = a.q_out + ((t0 + tok) * a.Hq + h) * D;
    } else {
      if (row < 0) return;
      const int hk = h - a.Hq - (is_v ? a.Hkv : 0);
      dst = (is_v ? a.v : a.k) + (row + (int64_t)hk * a.at.page) * D;
    }
    *(uint4*)(dst + 8 * lane) = y0;
    *(uint4*)(dst + D / 2 + 8 * lane) = y1;
  };
  for (int it = mine; it - mine < items; it += 2 * PASS) {  // the next share is on its way while one is worked on
    request(odd, it + PASS);
    process(even, it);
    if (it - mine + PASS >= items) break;
    request(even, it + 2 * PASS);
    process(odd, it + PASS);
  }
}

}  // namespace

int k_rope_paged(strictb200_ctx* ctx, const PagedRopeArgs& a) {
  Rates r;
  for (int i = 0; i < 64; i++) r.turn[i] = i < a.D / 2 ? std::pow((double)a.theta, -2.0 * i / a.D) / (2.0 * M_PI) : 0.0;
  // blocks for every SM first, then longer ones
  const int tokens = (int)std::max<int64_t>(1, std::min<int64_t>(MAX_TOKENS, (a.at.T + 4 * ctx->sm_count - 1) / (4 * ctx->sm_count)));
  const dim3 grid((unsigned)((a.at.T + tokens - 1) / tokens));
  SB_CUDA(sb_launch(ctx, a.D == 128 ? rope_paged_kernel<128> : rope_paged_kernel<64>, grid, dim3(THREADS), 0, a, r, tokens));
  ctx->launches++;
  return STRICTB200_OK;
}
