// Softmax attention of new tokens over a paged cache, grouped heads of 64 or 128 dims, bf16.
//
// One new token per sequence and at most 16 query heads per key/value head: the kernel here. Otherwise attention_paged_tc.cu.
#include <algorithm>

#include "mma_tiles.cuh"
#include "attention_paged.cuh"

using namespace mt;

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// ------------------------------------------------------------------ one new token per sequence
// Bound by HBM: every key and value is read once. A block is one key/value head of one sequence and a share of its key tiles; the G query heads of
// the key/value head are the rows of the products (mma.sync m16n8k16, 16 rows), warp w owns keys 16 w .. 16 w + 15 of every tile of 64 with a softmax
// of its own, and the four warps are joined at the end. Tiles come by cp.async into two stages; page numbers are fetched one piece of the walk (CT tiles) at
// a time. Positions that the row does not see, or whose entry names no page, are zeros in the tiles and -inf among the scores, so nothing that lies there counts.
//
// Shares: chunk c of CT tiles belongs to block c % gridDim.x, however long the sequence turns out to be. JOIN: 0 there is one block, 1 the
// blocks leave (maximum, sum, unnormalised output) in scratch for attn_paged_join_kernel, 2 they are one cluster and join through distributed shared memory.
constexpr int KT = 64;
constexpr int CT = 64;  // tiles of a piece at most: 1 KB of page numbers
constexpr int STAGES = 2;
enum { JOIN_NONE = 0, JOIN_SCRATCH = 1, JOIN_CLUSTER = 2 };
constexpr int CLUSTER_MAX = 8;

__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

template <int HD, int JOIN>
__global__ void __launch_bounds__(128) attn_paged_decode_kernel(PagedAttnArgs a, PagedJoin join, int ct) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int page_s[CT * 4];
  pdl_wait();
  pdl_trigger();
  const int part = blockIdx.x, parts = gridDim.x, hk = blockIdx.y, b = blockIdx.z;
  const int G = a.Hq / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3, mi = lane >> 3, r8 = lane & 7;
  const int64_t t0 = a.at.starts[b];
  const bool real = t0 >= 0 && t0 < a.at.T && a.at.starts[b + 1] > t0;  // the same for every block of a cluster
  if (!real) return;
  const int len = a.at.lens[b], pos = len - a.at.starts[b + 1] + (int)t0;
  const PagedWalk w = paged_walk(a.at, len, pos, pos, a.window, a.first, KT);
  const int lo = a.window ? max(0, pos - a.window + 1) : 0;
  const uint32_t sK = smem_u32(smem), sV = sK + STAGES * KT * 2 * HD;
  const int gp = a.at.page < KT ? KT / a.at.page : 1, gshift = a.at.page < KT ? a.at.shift : 6;  // pages of a tile; slots of a tile in one page

  uint32_t qf[HD / 16][4];
  {
    const bf16* q0 = a.q + (t0 * a.Hq + hk * G) * HD;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ks++) {
      const int d0 = ks * 16 + 2 * tig;
      qf[ks][0] = g < G ? *(const uint32_t*)(q0 + g * HD + d0) : 0u;
      qf[ks][1] = g + 8 < G ? *(const uint32_t*)(q0 + (g + 8) * HD + d0) : 0u;
      qf[ks][2] = g < G ? *(const uint32_t*)(q0 + g * HD + d0 + 8) : 0u;
      qf[ks][3] = g + 8 < G ? *(const uint32_t*)(q0 + (g + 8) * HD + d0 + 8) : 0u;
    }
  }
  float o[HD / 8][4];
#pragma unroll
  for (int j = 0; j < HD / 8; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[j][i] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  const float scale_log2 = a.scale * LOG2E;
  auto seen = [&](int j) { return j < w.end && (j >= lo || j < a.first); };

  for (int c0 = part * ct; c0 < w.total; c0 += parts * ct) {
    const int n = min(ct, w.total - c0);
    for (int i = threadIdx.x; i < n * gp; i += 128) page_s[i] = paged_page(a.at, b, (w.tile(c0 + i / gp) * KT + ((i % gp) << gshift)) >> a.at.shift);
    __syncthreads();
    auto load = [&](int t) {
      const int j0 = w.tile(c0 + t) * KT;
      constexpr int CH = HD / 8, RS = 128 / CH;  // 16-byte chunks of a row; rows that the block fetches at a time
      const int cc = threadIdx.x % CH, r0 = threadIdx.x / CH;
      const uint32_t st = (uint32_t)((t % STAGES) * KT * 2 * HD);
#pragma unroll
      for (int i = 0; i < KT / RS; i++) {
        const int r = r0 + i * RS, p = page_s[t * gp + (r >> gshift)];
        const bool ok = p >= 0 && seen(j0 + r);
        const int64_t at = ok ? ((p * (int64_t)a.Hkv + hk) * a.at.page + ((j0 + r) & (a.at.page - 1))) * HD + cc * 8 : 0;
        cp_async16(sK + st + tile_off<HD>(r, cc), a.k + at, ok);
        cp_async16(sV + st + tile_off<HD>(r, cc), a.v + at, ok);
      }
    };
    load(0);
    cp_async_commit();
    for (int t = 0; t < n; t++) {
      if (t + 1 < n) load(t + 1);
      cp_async_commit();
      cp_async_wait<1>();
      __syncthreads();
      const uint32_t tK = sK + (t % STAGES) * KT * 2 * HD, tV = sV + (t % STAGES) * KT * 2 * HD;
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < HD / 16; ks++) {
        uint32_t kb[4];
        ldsm_x4(tK + tile_off<HD>(warp * 16 + (mi >> 1) * 8 + r8, 2 * ks + (mi & 1)), kb);
        mma_bf16(s[0], qf[ks], kb[0], kb[1]);
        mma_bf16(s[1], qf[ks], kb[2], kb[3]);
      }
      const int r0 = warp * 16 + 2 * tig, j0 = w.tile(c0 + t) * KT;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = r0 + 8 * j + (i & 1);
          const float v = seen(j0 + r) && page_s[t * gp + (r >> gshift)] >= 0 ? s[j][i] * scale_log2 : -INFINITY;
          s[j][i] = v;
          mx[i >> 1] = fmaxf(mx[i >> 1], v);
        }
      float corr[2], m_use[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float m_new = fmaxf(m_run[r], mx[r]);
        m_use[r] = m_new == -INFINITY ? 0.f : m_new;
        corr[r] = exp2f(m_run[r] - m_use[r]);
        m_run[r] = m_new;
      }
      uint32_t pf[4], pl[4];
      {
        float p[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          p[j][0] = exp2f(s[j][0] - m_use[0]); p[j][1] = exp2f(s[j][1] - m_use[0]);
          p[j][2] = exp2f(s[j][2] - m_use[1]); p[j][3] = exp2f(s[j][3] - m_use[1]);
        }
        l_run[0] = l_run[0] * corr[0] + (p[0][0] + p[0][1] + p[1][0] + p[1][1]);
        l_run[1] = l_run[1] * corr[1] + (p[0][2] + p[0][3] + p[1][2] + p[1][3]);
        split_bf16(p[0][0], p[0][1], pf[0], pl[0]); split_bf16(p[0][2], p[0][3], pf[1], pl[1]);
        split_bf16(p[1][0], p[1][1], pf[2], pl[2]); split_bf16(p[1][2], p[1][3], pf[3], pl[3]);
      }
#pragma unroll
      for (int j = 0; j < HD / 8; j++) {
        o[j][0] *= corr[0]; o[j][1] *= corr[0];
        o[j][2] *= corr[1]; o[j][3] *= corr[1];
      }
#pragma unroll
      for (int jj = 0; jj < HD / 16; jj++) {
        uint32_t vb[4];
        ldsm_x4_t(tV + tile_off<HD>(warp * 16 + (mi & 1) * 8 + r8, 2 * jj + (mi >> 1)), vb);
        mma_bf16(o[2 * jj], pf, vb[0], vb[1]);
        mma_bf16(o[2 * jj + 1], pf, vb[2], vb[3]);
        mma_bf16(o[2 * jj], pl, vb[0], vb[1]);
        mma_bf16(o[2 * jj + 1], pl, vb[2], vb[3]);
      }
      __syncthreads();
    }
    cp_async_wait<0>();
  }
#pragma unroll
  for (int r = 0; r < 2; r++) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
  }
  // the four warps joined through shared memory (the tiles are free after the last barrier)
  float* so = (float*)smem;                    // [4 warps][16 rows][HD]
  float2* sml = (float2*)(so + 4 * 16 * HD);   // [4 warps][16 rows]
  float* jo = (float*)(sml + 4 * 16);          // [G][HD] joined
  float2* jml = (float2*)(jo + 16 * HD);       // [G]
#pragma unroll
  for (int r = 0; r < 2; r++) {
    const int row = g + 8 * r;
    if (row < G) {
#pragma unroll
      for (int j = 0; j < HD / 8; j++) *(float2*)(so + (warp * 16 + row) * HD + 8 * j + 2 * tig) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
      if (tig == 0) sml[warp * 16 + row] = make_float2(m_run[r], l_run[r]);
    }
  }
  __syncthreads();
  bf16* out = a.out + (t0 * a.Hq + hk * G) * HD;
  for (int e = threadIdx.x; e < G * (HD / 4); e += 128) {
    const int row = e / (HD / 4), d = e % (HD / 4) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) M = fmaxf(M, sml[i * 16 + row].x);
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float f = weight_of(sml[i * 16 + row].x, M);
      const float4 p = *(const float4*)(so + (i * 16 + row) * HD + d);
      L += sml[i * 16 + row].y * f;
      O.x += p.x * f; O.y += p.y * f; O.z += p.z * f; O.w += p.w * f;
    }
    if (JOIN == JOIN_NONE) {
      const float inv = L == 0.f ? 0.f : 1.0f / L;
      *(uint2*)(out + row * HD + d) = make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
    } else if (JOIN == JOIN_SCRATCH) {
      const int64_t at = (t0 * a.Hq + hk * G + row) * parts + part;
      if (L != 0.f) *(float4*)(join.o + at * HD + d) = O;  // read only where the sum is not zero
      if (d == 0) join.ml[at] = make_float2(M, L);
    } else {
      *(float4*)(jo + row * HD + d) = O;
      if (d == 0) jml[row] = make_float2(M, L);
    }
  }
  if (JOIN == JOIN_CLUSTER) {
    __syncthreads();  // .aligned: every warp at once
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    auto remote = [](uint32_t local, int rank) {
      uint32_t x;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(x) : "r"(local), "r"(rank));
      return x;
    };
    for (int e = part * 128 + threadIdx.x; e < G * (HD / 4); e += parts * 128) {
      const int row = e / (HD / 4), d = e % (HD / 4) * 4;
      float2 ml[CLUSTER_MAX];
      float4 p[CLUSTER_MAX];
#pragma unroll
      for (int i = 0; i < CLUSTER_MAX; i++)
        if (i < parts) {
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[i].x), "=f"(ml[i].y) : "r"(remote(smem_u32(jml + row), i)) : "memory");
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(p[i].x), "=f"(p[i].y), "=f"(p[i].z), "=f"(p[i].w)
                       : "r"(remote(smem_u32(jo + row * HD + d), i))
                       : "memory");
        }
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int i = 0; i < CLUSTER_MAX; i++)
        if (i < parts) M = fmaxf(M, ml[i].x);
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < CLUSTER_MAX; i++)
        if (i < parts) {
          const float f = weight_of(ml[i].x, M);
          L += ml[i].y * f;
          O.x += p[i].x * f; O.y += p[i].y * f; O.z += p[i].z * f; O.w += p[i].w * f;
        }
      const float inv = L == 0.f ? 0.f : 1.0f / L;
      *(uint2*)(out + row * HD + d) = make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
    }
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // nobody leaves while its memory is read
  }
}

// A warp per row and head: out = sum_i w_i o_i / sum_i w_i l_i over the parts, w_i = 2^(m_i - max).
template <int HD>
__global__ void __launch_bounds__(256) attn_paged_join_kernel(PagedAttnArgs a, PagedJoin join) {
  constexpr int E = HD / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  if (at >= a.at.T * a.Hq) return;
  const int64_t t = at / a.Hq;
  if (t < a.at.starts[0] || t >= a.at.starts[a.at.B]) return;
  const float2* ml = join.ml + at * join.parts;
  float M = -INFINITY, L = 0.f, O[E];
  for (int i = lane; i < join.parts; i += 32) M = fmaxf(M, ml[i].x);
  M = warp_max(M);
#pragma unroll
  for (int e = 0; e < E; e++) O[e] = 0.f;
  for (int i = 0; i < join.parts; i++) {
    const float2 v = ml[i];
    if (v.y == 0.f) continue;
    const float f = weight_of(v.x, M);
    L += v.y * f;
    const float* o = join.o + (at * join.parts + i) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) O[e] += o[e] * f;
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
  for (int e = 0; e < E; e += 2) *(uint32_t*)(a.out + at * HD + lane * E + e) = pack_bf16(O[e] * inv, O[e + 1] * inv);
}

template <int HD>
int decode(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  const size_t tiles_bytes = (size_t)2 * STAGES * KT * 2 * HD, join_bytes = (size_t)(5 * 16 * HD) * 4 + 5 * 16 * 8;
  const size_t smem = std::max(tiles_bytes, join_bytes);
  static SbDeviceOnce once;
  SB_CUDA(once.run(ctx->device, [&] {
    for (auto f : {attn_paged_decode_kernel<HD, JOIN_NONE>, attn_paged_decode_kernel<HD, JOIN_SCRATCH>, attn_paged_decode_kernel<HD, JOIN_CLUSTER>}) {
      cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }));
  const int64_t tiles = std::max<int64_t>(1, paged_walk_tiles(a, KT)), units = (int64_t)a.at.B * a.Hkv, slots = (int64_t)ctx->sm_count * 3;
  // One wave: as many parts as there are places, in a cluster of at most eight where that leaves a block few tiles. Several waves: pieces of at least
  // eight tiles, four waves of them if the sequences are as long as they may be, so that uneven lengths even out.
  int64_t parts = std::min(tiles, slots / units);
  int join = JOIN_CLUSTER;
  if (units * 2 > slots) {
    parts = std::max<int64_t>(1, std::min(tiles / 8, (4 * slots + units - 1) / units));
    join = JOIN_SCRATCH;
  } else if (parts > CLUSTER_MAX) {
    if (tiles <= CLUSTER_MAX * 4) parts = CLUSTER_MAX;
    else {
      parts = std::min<int64_t>(parts, (tiles + 1) / 2);
      join = JOIN_SCRATCH;
    }
  }
  parts = std::min<int64_t>(parts, 256);
  if (parts <= 1) join = JOIN_NONE, parts = 1;
  const int ct = (int)std::min<int64_t>(CT, (tiles + parts - 1) / parts);
  const dim3 grid((unsigned)parts, (unsigned)a.Hkv, (unsigned)a.at.B);
  PagedJoin buf{};
  buf.parts = (int)parts;
  if (join == JOIN_SCRATCH) SB_TRY(paged_join_scratch(ctx, a, (int)parts, &buf));
  if (join == JOIN_NONE) SB_CUDA(sb_launch(ctx, attn_paged_decode_kernel<HD, JOIN_NONE>, grid, dim3(128), smem, a, buf, ct));
  else if (join == JOIN_SCRATCH) SB_CUDA(sb_launch(ctx, attn_paged_decode_kernel<HD, JOIN_SCRATCH>, grid, dim3(128), smem, a, buf, ct));
  else SB_CUDA(sb_launch_cluster(ctx, attn_paged_decode_kernel<HD, JOIN_CLUSTER>, grid, dim3(128), smem, dim3((unsigned)parts), a, buf, ct));
  ctx->launches++;
  return join == JOIN_SCRATCH ? paged_join(ctx, a, buf) : STRICTB200_OK;
}

}  // namespace

int paged_join_scratch(strictb200_ctx* ctx, const PagedAttnArgs& a, int parts, PagedJoin* join) {
  const size_t rows = (size_t)a.at.T * a.Hq * parts;
  void* ws;
  SB_TRY(sb_ws(ctx, rows * (a.D * sizeof(float) + sizeof(float2)), &ws));
  join->o = (float*)ws;
  join->ml = (float2*)((float*)ws + rows * a.D);
  join->parts = parts;
  return STRICTB200_OK;
}
int paged_join(strictb200_ctx* ctx, const PagedAttnArgs& a, const PagedJoin& join) {
  const dim3 grid((unsigned)((a.at.T * a.Hq + 7) / 8));
  SB_CUDA(sb_launch(ctx, a.D == 128 ? attn_paged_join_kernel<128> : attn_paged_join_kernel<64>, grid, dim3(256), 0, a, join));
  ctx->launches++;
  return STRICTB200_OK;
}
int64_t paged_walk_tiles(const PagedAttnArgs& a, int kt) {
  const int64_t len = std::min<int64_t>(a.max_len, (int64_t)a.at.ld << a.at.shift), tiles = (len + kt - 1) / kt;
  if (!a.window) return tiles;
  return std::min<int64_t>(tiles, ((int64_t)a.window + a.max_new) / kt + 2 + ((int64_t)a.first + kt - 1) / kt);
}

int k_attn_paged(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  if (a.max_new > 1 || a.Hq / a.Hkv > 16 || a.at.B > 65535) return k_attn_paged_tiles(ctx, a);
  return a.D == 128 ? decode<128>(ctx, a) : decode<64>(ctx, a);
}
