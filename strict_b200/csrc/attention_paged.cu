// Softmax attention of new tokens over a paged cache, grouped heads of 64 or 128 dims, bf16.
//
// Few rows, where a row is one query head of one new token: at most 16 per sequence and key/value head. More: attention_paged_tc.cu.
#include <algorithm>
#include <cmath>

#include "mma_tiles.cuh"
#include "attention_paged.cuh"

using namespace mt;

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// Bound by HBM: every key and value is read once (64 sequences of 1 to 16 thousand keys, 2.28 GB: 339 us, 6.7 TB/s; times in these files are
// of calls in a row on the same data, 352 us with other data between them). A block is one key/value head of one sequence and a share of its tiles of 64 keys. The last warp copies:
// its lanes look the pages up, well ahead, and request the tile by TMA (boxes of min(page, 64) keys x 64 dims, 128-byte swizzle) into a ring
// of `stages`. The others have 16 keys of every tile and all 8 NB rows each, with a softmax of their own; the four shares of the keys are
// joined at the end.
// Products are mma.sync m16n8k16 with keys (then dims) as the 16 rows and attention rows as the 8 columns, S^T = K Q^T and O^T = V^T P^T: at most eight
// rows waste nothing that way. (With the rows as rows, half of everything was idle: 874 instructions per warp and tile, 166 registers and 5.3 TB/s.)
// Positions that a row does not see, or whose entry names no page, are not fetched or hidden by index: their scores become -inf, and where some row
// does not see some of the 16 keys, values that are not finite are replaced by zeros on their way into the product (add_poison has the rest), so nothing
// that lies there counts.
//
// Shares: piece c of ct tiles belongs to block c % gridDim.x, however long the sequence turns out to be. JOIN: 0 there is one block, 1 the
// blocks leave (maximum, sum, unnormalised output) in scratch for attn_paged_join_kernel, 2 they are one cluster and join through distributed shared memory.
constexpr int KT = 64;
constexpr int MAX_STAGES = 6;
// Up to here this kernel, beyond it attention_paged_tc.cu: 64 sequences of 1 to 16 thousand keys with 16 rows take 332 us here and 417 there, 16 equal ones of 8
// thousand with 12 rows 105 and 135 (uneven ones 93 and 84).
constexpr int FEW_ROWS = 16;
enum { JOIN_NONE = 0, JOIN_SCRATCH = 1, JOIN_CLUSTER = 2 };
constexpr int CLUSTER_MAX = 8;

__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

constexpr size_t few_tile_bytes(int HD) { return (size_t)KT * 2 * HD; }
constexpr size_t few_smem(int HD, int rows, int stages) {
  const size_t ring = 2 * stages * few_tile_bytes(HD), join = (size_t)rows * ((4 * (HD + 4) + HD) * 4 + 5 * 8);
  return (ring > join ? ring : join) + 1024;
}

// blocks that fit on an SM: shared memory of two stages (8 rows of 128 dims), registers (otherwise)
template <int HD, int NB>
constexpr int few_fit() { return NB == 2 ? (HD == 128 ? 2 : 3) : HD == 128 ? 3 : 4; }

template <int HD, int NB, int JOIN>
__global__ void __launch_bounds__(160, few_fit<HD, NB>()) attn_paged_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                       const __grid_constant__ PagedAttnArgs a, PagedJoin join, int ct, int stages, int* status) {
  constexpr int ATOM = KT * 128, TILE = ATOM * (HD / 64);  // bytes of 64 keys x 64 dims, and of a tile
  constexpr int WARPS = 4, ROWS = 8 * NB, BLOCK = 32 * (WARPS + 1);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  __shared__ uint32_t page_bits[MAX_STAGES];
  __shared__ Poison poison;
  const int part = blockIdx.x, parts = gridDim.x, hk = blockIdx.y, b = blockIdx.z;
  const int G = a.Hq / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3, mi = lane >> 3, r8 = lane & 7;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; i++) {
      tc::mbar_init(smem_u32(&full[i]), 1);
      tc::mbar_init(smem_u32(&empty[i]), WARPS);
    }
    poison.n = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int box = min(a.at.page, KT), boxes = KT / box;
  const int64_t t0 = a.at.starts[b];
  const int last = a.at.starts[b + 1], len = a.at.lens[b];
  if (t0 < 0 || last > a.at.T || last <= t0) return;  // the same for every block of a cluster
  const int R = (int)min((int64_t)ROWS / G, last - t0) * G, lo_pos = len - last + (int)t0, hi_pos = lo_pos + R / G - 1;
  const int lo_key = window_begin(lo_pos, a.window);
  const PagedWalk w = paged_walk(a.at, len, lo_key, hi_pos, a.first, KT);
  const int n = share_count(w.total, part, parts, ct);
  const uint32_t sK = smem_u32(smem), sV = sK + stages * TILE;
  auto row_head = [&](int row) { return (t0 + row / G) * a.Hq + hk * G + row % G; };  // place among all rows and heads

  float o[HD / 16][NB][4], m_run[NB][2], l_run[NB][2];
  const int kg = warp & 3;  // keys 16 kg .. of a tile
  if (warp == WARPS) {
    auto page_of = [&](int i, int x) {
      const int j = i < n ? w.tile(share_tile(i, part, parts, ct)) * KT + x * box : w.end;
      return j < w.end ? paged_page(a.at, b, j >> a.at.shift) : -1;
    };
    PageNames names;
    names.begin(boxes, lane, page_of);
    int got = 0;
    bool good = true;
    int st = 0;
    uint32_t ph = 1;  // of the round in front
    for (int i = 0; i < n; i++) {
      const int page = names.of(i, boxes, lane, page_of);
      const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
      const int j = w.tile(share_tile(i, part, parts, ct)) * KT + lane * box;
      const int row = page < 0 ? 0 : (int)((page * (int64_t)a.Hkv + hk) * a.at.page) + (j & (a.at.page - 1));
      if (i >= stages) good = tc::mbar_wait(smem_u32(&empty[st]), ph);
      if (!__all_sync(0xffffffffu, good)) {
        if (lane == 0) tc::set_status(status, 47);
        break;
      }
      if (lane == 0) {
        page_bits[st] = there;
        tc::mbar_expect_tx(smem_u32(&full[st]), (uint32_t)(__popc(there) * box * 2 * 2 * HD));
      }
      __syncwarp();
      if (page >= 0)
#pragma unroll
        for (int x = 0; x < HD / 64; x++) {
          tc::tma_load_2d(sK + st * TILE + x * ATOM + lane * box * 128, &map_k, x * 64, row, smem_u32(&full[st]));
          tc::tma_load_2d(sV + st * TILE + x * ATOM + lane * box * 128, &map_v, x * 64, row, smem_u32(&full[st]));
        }
      got = i + 1;
      if (++st == stages) st = 0, ph ^= 1;
    }
    // copies in flight have landed before this block's memory is somebody else's; only needed where a wait gave up
    for (int i = max(0, got - stages); i < got; i++) tc::mbar_wait(smem_u32(&full[i % stages]), (uint32_t)((i / stages) & 1));
    __syncwarp();
  } else {
    // queries as columns: row 8 nb + g, dims 16 ks + 2 tig ..
    uint32_t qf[HD / 16][NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int row = 8 * nb + g;
      const bf16* q = a.q + (row < R ? row_head(row) * HD : 0) + 2 * tig;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ks++) {
        qf[ks][nb][0] = row < R ? *(const uint32_t*)(q + ks * 16) : 0u;
        qf[ks][nb][1] = row < R ? *(const uint32_t*)(q + ks * 16 + 8) : 0u;
      }
    }
    int pos[NB][2];  // of the columns that this thread has scores of
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
      for (int j = 0; j < HD / 16; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[j][nb][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        m_run[nb][h] = -INFINITY;
        l_run[nb][h] = 0.f;
        pos[nb][h] = lo_pos + (8 * nb + 2 * tig + h) / G;
      }
    }
    const float scale_log2 = a.scale * LOG2E;
    const uint32_t sw = (uint32_t)r8 << 4;  // chunk c of row r lies at chunk c ^ (r & 7)
    bool ok = true;
    int st = 0, step = part * ct, left = ct;  // place in the walk, tiles of the piece
    uint32_t ph = 0;
    for (int i = 0; i < n; i++) {
      const int j0 = w.tile(step++) * KT + kg * 16;
      if (--left == 0) left = ct, step += (parts - 1) * ct;
      ok = ok && tc::mbar_wait(smem_u32(&full[st]), ph);
      __syncwarp();
      const uint32_t tK = sK + st * TILE + kg * 16 * 128, tV = sV + st * TILE + kg * 16 * 128;
      const bool there = page_bits[st] >> (kg * 16 / box) & 1;
      const bool whole = there && sees_all(a, w.end, j0, 16, lo_pos, hi_pos);
      // values that some row may see: what lies behind them, or where nothing was fetched (the last sums of an earlier block, say), is not looked for again
      uint32_t seen[2] = {0, 0};
      if (there && !whole) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = j0 + (e >> 1) * 8 + 2 * tig + (e & 1);
          if (j < w.end && (j >= lo_key || j < a.first)) seen[e >> 1] |= e & 1 ? 0xFFFF0000u : 0xFFFFu;
        }
      }
      // scores: keys g and g + 8, rows 2 tig and 2 tig + 1
      float s[NB][4], s2[NB][4];  // two sums, so that half as many products wait for one another
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[nb][e] = s2[nb][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ks++) {
        uint32_t kf[4];
        ldsm_x4(tK + (ks >> 2) * ATOM + ((mi & 1) * 8 + r8) * 128 + ((((ks & 3) * 2 + (mi >> 1)) << 4) ^ sw), kf);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) mma_bf16(ks & 1 ? s2[nb] : s[nb], kf, qf[ks][nb][0], qf[ks][nb][1]);
      }
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[nb][e] += s2[nb][e];
      if (!whole) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int j = j0 + g + (e & 2) * 4, p = pos[nb][e & 1];
            if (!(there && j <= p && j < w.end && (!a.window || j > p - a.window || j < a.first))) s[nb][e] = -INFINITY;
          }
      }
      uint32_t pf[NB][2], pl[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        float mx[2] = {fmaxf(s[nb][0], s[nb][2]), fmaxf(s[nb][1], s[nb][3])}, corr[2], base[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 4));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 8));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 16));
          const float m_new = fmaxf(m_run[nb][h], mx[h] * scale_log2);
          base[h] = m_new == -INFINITY ? 0.f : -m_new;
          corr[h] = tc::ex2_approx(m_run[nb][h] + base[h]);
          m_run[nb][h] = m_new;
        }
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = tc::ex2_approx(fmaf(s[nb][e], scale_log2, base[e & 1]));
        l_run[nb][0] = l_run[nb][0] * corr[0] + (p[0] + p[2]);
        l_run[nb][1] = l_run[nb][1] * corr[1] + (p[1] + p[3]);
        split_bf16(p[0], p[1], pf[nb][0], pl[nb][0]);
        split_bf16(p[2], p[3], pf[nb][1], pl[nb][1]);
#pragma unroll
        for (int x = 0; x < 2; x++) {
          pf[nb][x] = transposed(pf[nb][x]);
          pl[nb][x] = transposed(pl[nb][x]);
        }
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
          for (int j = 0; j < HD / 16; j++) {
            o[j][nb][0] *= corr[0]; o[j][nb][1] *= corr[1];
            o[j][nb][2] *= corr[0]; o[j][nb][3] *= corr[1];
          }
        }
      }
#pragma unroll
      for (int j4 = 0; j4 < HD / 16; j4 += 4) {
        uint32_t vf[4][4];  // dims 16 j .. as rows, keys as columns; four products between the two that add to one sum
#pragma unroll
        for (int j = 0; j < 4; j++) ldsm_x4_t(tV + (j4 >> 2) * ATOM + ((mi >> 1) * 8 + r8) * 128 + (((j * 2 + (mi & 1)) << 4) ^ sw), vf[j]);
        if (!whole) {
          uint32_t found = 0;
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
              found |= not_finite(vf[j][x] & seen[x >> 1]);  // this thread's keys are j0 + 8 (x / 2) + 2 tig and the next one
              vf[j][x] = only_finite(vf[j][x]);
            }
          if (__any_sync(0xffffffffu, found != 0) && lane == 0) note_poison(poison, i);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int nb = 0; nb < NB; nb++) mma_bf16(o[j4 + j][nb], vf[j], pf[nb][0], pf[nb][1]);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int nb = 0; nb < NB; nb++) mma_bf16(o[j4 + j][nb], vf[j], pl[nb][0], pl[nb][1]);
      }
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[st])) : "memory");
      if (++st == stages) st = 0, ph ^= 1;
    }
    if (!__all_sync(0xffffffffu, ok) && lane == 0) tc::set_status(status, 48);
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l_run[nb][h] += __shfl_xor_sync(0xffffffffu, l_run[nb][h], x);
  }
  __syncthreads();  // every copy has been waited for, and nobody reads a tile any more
  // the four shares of the keys joined through shared memory
  constexpr int LD = HD + 4;
  float* so = (float*)smem;                    // [4][ROWS][LD]
  float* jo = so + 4 * ROWS * LD;              // [ROWS][HD] joined
  float2* sml = (float2*)(jo + ROWS * HD);     // [4][ROWS]
  float2* jml = sml + 4 * ROWS;                // [ROWS]
  if (warp < WARPS) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = 8 * nb + 2 * tig + h;
        if (row < R) {
#pragma unroll
          for (int j = 0; j < HD / 16; j++) {
            so[(kg * ROWS + row) * LD + 16 * j + g] = o[j][nb][h];
            so[(kg * ROWS + row) * LD + 16 * j + g + 8] = o[j][nb][2 + h];
          }
          if (g == 0) sml[kg * ROWS + row] = make_float2(m_run[nb][h], l_run[nb][h]);
        }
      }
  }
  __syncthreads();
  const bool bad = poison.n > 0;
  for (int e = threadIdx.x; e < R * (HD / 4); e += BLOCK) {
    const int row = e / (HD / 4), d = e % (HD / 4) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) M = fmaxf(M, sml[i * ROWS + row].x);
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float f = weight_of(sml[i * ROWS + row].x, M);
      const float4 p = *(const float4*)(so + (i * ROWS + row) * LD + d);
      L += sml[i * ROWS + row].y * f;
      O.x += p.x * f; O.y += p.y * f; O.z += p.z * f; O.w += p.w * f;
    }
    if (bad && L != 0.f) {
      float r[4] = {O.x, O.y, O.z, O.w};
      add_poison(a, w, b, hk, part, parts, ct, KT, 16, lo_pos, hi_pos, poison, 0, 1, n, lo_pos + row / G, d, 4, r);
      O = make_float4(r[0], r[1], r[2], r[3]);
    }
    if (JOIN == JOIN_NONE) {
      const float inv = L == 0.f ? 0.f : 1.0f / L;
      *(uint2*)(a.out + row_head(row) * HD + d) = make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
    } else if (JOIN == JOIN_SCRATCH) {
      const int64_t at = row_head(row) * parts + part;
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
    for (int e = part * BLOCK + threadIdx.x; e < R * (HD / 4); e += parts * BLOCK) {
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
      *(uint2*)(a.out + row_head(row) * HD + d) = make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
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
  const float* o = join.o + at * join.parts * HD + lane * E;
  float M = -INFINITY, L = 0.f, O[E];
  for (int i = lane; i < join.parts; i += 32) M = fmaxf(M, ml[i].x);
  M = warp_max(M);
#pragma unroll
  for (int e = 0; e < E; e++) O[e] = 0.f;
  for (int i0 = 0; i0 < join.parts; i0 += 32) {  // a lane has the weight of a part; the outputs of eight parts are requested together
    const float2 v = i0 + lane < join.parts ? ml[i0 + lane] : make_float2(-INFINITY, 0.f);
    const float f = weight_of(v.x, M);
    L += v.y * f;
    const unsigned there = __ballot_sync(0xffffffffu, v.y != 0.f);
    for (int i = 0; i < min(32, join.parts - i0); i += 8) {
      float x[8][E];
#pragma unroll
      for (int n = 0; n < 8; n++)
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 y = there >> (i + n) & 1 ? *(const float2*)(o + (int64_t)(i0 + i + n) * HD + e) : make_float2(0.f, 0.f);
          x[n][e] = y.x;
          x[n][e + 1] = y.y;
        }
#pragma unroll
      for (int n = 0; n < 8; n++) {
        const float fn = __shfl_sync(0xffffffffu, f, i + n);
#pragma unroll
        for (int e = 0; e < E; e++)
          if (there >> (i + n) & 1) O[e] += x[n][e] * fn;
      }
    }
  }
  L = warp_sum(L);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
  for (int e = 0; e < E; e += 2) *(uint32_t*)(a.out + at * HD + lane * E + e) = pack_bf16(O[e] * inv, O[e + 1] * inv);
}

struct FewPlan {
  int parts = 1, stages = 2, join = JOIN_NONE;
};
// How the keys are cut, from the sizes, by a model in microseconds. A tile costs a block `tile` times the blocks on its SM (an SM's share of HBM, 46 GB/s), but
// at least `chain` (its products and its softmax one after the other) and 1.3 / stages (the latency of a copy); starting and ending, 3 for the first blocks,
// 7 for every further round of them; the join in a cluster 1.5, the one through scratch 4 and its bytes. Only the longest sequence's length is known here, and the
// blocks of a shorter one that have no tile leave at once. So a cut is costed twice, for sequences that are all as long and for lengths spread
// below that one (mean 0.65, and half a block more per unit that is not full), and the sum counts: 16 sequences of 5 to 8 thousand keys, two new tokens and eight
// heads took 79 us in the two parts that suit equal lengths, 61 in four.
// Ring: what shared memory leaves the blocks that share an SM. Clusters need all their blocks at once: one round only, counted with 7/8 of the SMs, and
// with shared memory for two blocks on each, or those that find no eight empty SMs wait for a second one.
FewPlan plan_few(const strictb200_ctx* ctx, int HD, int fit, double chain, int64_t B, int64_t units, int64_t tiles, double out_floats) {
  const double stage = 2.0 * few_tile_bytes(HD), tile = stage / 46e3, sms = ctx->sm_count, slots = fit * sms;
  auto ring = [&](int share) { return (int)((double)(220 << 10) / share / stage - 0.1); };
  FewPlan best;
  double best_us = 1e30;
  for (int64_t parts = 1; parts <= std::min<int64_t>(tiles, 128); parts += parts < 16 ? 1 : parts / 4) {
    if (parts > 1 && out_floats * parts * 4 > (double)(512 << 20)) break;  // scratch
    const double ct = (double)((tiles + parts - 1) / parts), blocks = (double)(units * parts);
    const bool cluster = parts > 1 && parts <= CLUSTER_MAX && blocks <= 0.875 * slots;
    FewPlan p;
    p.parts = (int)parts;
    p.join = parts == 1 ? JOIN_NONE : cluster ? JOIN_CLUSTER : JOIN_SCRATCH;
    const int share = blocks <= slots ? std::max(cluster ? 2 : 1, (int)std::ceil(blocks / sms)) : parts == 1 ? 2 : fit;
    p.stages = std::max(2, std::min<int>({MAX_STAGES, (int)ct, ring(share)}));
    const double alone = std::max(chain, 1.3 / p.stages);
    auto round = [&](double n) { return n > 0 ? ct * std::max(tile * std::ceil(n / sms), alone) : 0; };  // of n blocks
    const double full = std::floor(blocks / slots);
    double us = full * round(slots) + round(blocks - full * slots) + 7 * blocks / slots;
    if (B > 1) {
      const double some = std::min(blocks, units * (0.65 * parts + 0.5)), work = units * tiles * 0.65 / sms * std::max(tile, alone / fit);
      us += some <= slots ? round(some) + 7 * some / slots : work + 0.25 * ct * chain * std::min(1.0, sms / some) + 7 * some / slots;
    } else {
      us *= 2;
    }
    us = us / 2 + (parts == 1 ? 0 : cluster ? 1.5 : 4 + out_floats * parts * 8 / 6e6);
    if (us < best_us * 0.97) best_us = us, best = p;
  }
  return best;
}

template <int HD, int NB>
int few_rows(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  static SbDeviceOnce once;
  SB_CUDA(once.run(ctx->device, [&] {
    for (auto f : {attn_paged_few_kernel<HD, NB, JOIN_NONE>, attn_paged_few_kernel<HD, NB, JOIN_SCRATCH>, attn_paged_few_kernel<HD, NB, JOIN_CLUSTER>}) {
      cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem(HD, 8 * NB, MAX_STAGES));
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }));
  const int64_t tiles = std::max<int64_t>(1, paged_walk_tiles(a, KT));
  const FewPlan plan = plan_few(ctx, HD, few_fit<HD, NB>(), (HD == 128 ? 0.8 : 0.6) * (NB == 2 ? 1.4 : 1), a.at.B, (int64_t)a.at.B * a.Hkv, tiles, (double)a.at.T * a.Hq * HD);
  const int parts = plan.parts, ct = (int)((tiles + parts - 1) / parts), stages = plan.stages;
  const size_t smem = few_smem(HD, 8 * NB, stages);
  const dim3 grid((unsigned)parts, (unsigned)a.Hkv, (unsigned)a.at.B);
  PagedJoin buf;
  if (plan.join == JOIN_SCRATCH) SB_TRY(paged_join_scratch(ctx, a, parts, &buf));
  CUtensorMap mk, mv;
  const int64_t rows = (int64_t)a.at.n_pages * a.Hkv * a.at.page;
  SB_TRY(paged_map_rows(&mk, a.k, rows, HD, std::min(a.at.page, KT)));
  SB_TRY(paged_map_rows(&mv, a.v, rows, HD, std::min(a.at.page, KT)));
  const dim3 block(160);
  if (plan.join == JOIN_NONE) SB_CUDA(sb_launch(ctx, attn_paged_few_kernel<HD, NB, JOIN_NONE>, grid, block, smem, mk, mv, a, buf, ct, stages, ctx->d_status));
  else if (plan.join == JOIN_SCRATCH) SB_CUDA(sb_launch(ctx, attn_paged_few_kernel<HD, NB, JOIN_SCRATCH>, grid, block, smem, mk, mv, a, buf, ct, stages, ctx->d_status));
  else SB_CUDA(sb_launch_cluster(ctx, attn_paged_few_kernel<HD, NB, JOIN_CLUSTER>, grid, block, smem, dim3((unsigned)parts), mk, mv, a, buf, ct, stages, ctx->d_status));
  ctx->launches++;
  return plan.join == JOIN_SCRATCH ? paged_join(ctx, a, buf) : STRICTB200_OK;
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
  const int64_t rows = (int64_t)std::max(1, a.max_new) * (a.Hq / a.Hkv);
  if (rows > FEW_ROWS || a.at.B > 65535) return k_attn_paged_tiles(ctx, a);
  if (rows > 8) return a.D == 128 ? few_rows<128, 2>(ctx, a) : few_rows<64, 2>(ctx, a);
  return a.D == 128 ? few_rows<128, 1>(ctx, a) : few_rows<64, 1>(ctx, a);
}
