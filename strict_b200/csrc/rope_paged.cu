// Norm and rotation of the new tokens' heads, keys and values into the pages of a cache.
#include <cmath>

#include "paged.cuh"

namespace {

struct Rates {
  double turn[64];  // theta^(-2i/D) / (2 pi): turns per position of the pair i
};

// A block per token, a warp per head at a time; a lane holds D / 32 neighbouring dims. The angles of the token are made once for all of its heads:
// position times rate in 64 bits, less the whole turns, sine and cosine of the rest in 32.
template <int D>
__global__ void __launch_bounds__(256) rope_paged_kernel(PagedRopeArgs a, const __grid_constant__ Rates r) {
  constexpr int E = D / 32;
  __shared__ float cos_s[D / 2], sin_s[D / 2];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = paged_seq(a.at, t);
  if (b >= a.at.B) return;
  const int pos = a.at.lens[b] - a.at.starts[b + 1] + (int)t;
  if (threadIdx.x < D / 2) {
    double x = pos * r.turn[threadIdx.x];
    x -= rint(x);
    sincospif(2.f * (float)x, &sin_s[threadIdx.x], &cos_s[threadIdx.x]);
  }
  const int page = pos >= 0 ? paged_page(a.at, b, pos >> a.at.shift) : -1;
  const int slot = pos & (a.at.page - 1);
  __syncthreads();
  for (int h = warp; h < a.Hq + 2 * a.Hkv; h += 8) {
    float x[E];
    for (int e = 0; e < E; e++) x[e] = __bfloat162float(a.qkv[(t * (a.Hq + 2 * a.Hkv) + h) * D + lane * E + e]);
    const bool is_v = h >= a.Hq + a.Hkv;
    if (!is_v) {
      const float* gain = h < a.Hq ? a.qgain : a.kgain;
      if (gain) {
        float ss = 0.f;
        for (int e = 0; e < E; e++) ss += x[e] * x[e];
        const float rr = 1.0f / sqrtf(warp_sum(ss) / D + a.eps);
        for (int e = 0; e < E; e++) x[e] *= rr * gain[lane * E + e];
      }
      for (int e = 0; e < E; e++) {
        const float other = __shfl_xor_sync(0xffffffffu, x[e], 16);
        const int i = (lane & 15) * E + e;
        x[e] = lane < 16 ? x[e] * cos_s[i] - other * sin_s[i] : x[e] * cos_s[i] + other * sin_s[i];
      }
    }
    bf16* dst = nullptr;
    if (h < a.Hq) dst = a.q_out + (t * a.Hq + h) * D;
    else if (page >= 0) dst = (is_v ? a.v : a.k) + ((page * (int64_t)a.Hkv + (h - a.Hq) % a.Hkv) * a.at.page + slot) * D;
    if (dst)
      for (int e = 0; e < E; e++) dst[lane * E + e] = __float2bfloat16_rn(x[e]);
  }
}

}  // namespace

int k_rope_paged(strictb200_ctx* ctx, const PagedRopeArgs& a) {
  Rates r;
  for (int i = 0; i < 64; i++) r.turn[i] = i < a.D / 2 ? std::pow((double)a.theta, -2.0 * i / a.D) / (2.0 * M_PI) : 0.0;
  if (a.D == 128) rope_paged_kernel<128><<<(unsigned)a.at.T, 256, 0, ctx->stream>>>(a, r);
  else rope_paged_kernel<64><<<(unsigned)a.at.T, 256, 0, ctx->stream>>>(a, r);
  SB_LAUNCHED(ctx);
  return STRICTB200_OK;
}
