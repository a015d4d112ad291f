// Softmax attention of new tokens over a paged cache on the tcgen05 tensor cores: drafted tokens, chunks and whole prompts.
//
// A row of the products is one query head of one new token: the G heads that share a key/value head are packed behind one another, 128 / G tokens to a
// tile of 128 rows (one TMA box: 64 dims x G heads x tokens), so keys and values are fetched once for all of them and a tile spans few positions. Rows
// are lanes of tensor memory. Per tile of 128 keys, as in the attention over contiguous caches:
//   S = Q K^T      operands in shared memory, fp32 sums in tensor memory
//   softmax        a thread per row, running maximum followed lazily (a row of O is rescaled when its maximum grew by more than 2^8), weights back to
//                  tensor memory as two bf16 terms (hi + lo by truncation: 2^-16)
//   O += P V       weights from tensor memory, values from shared memory; O stays in tensor memory
// Roles: warps 0..7 softmax, 8 issues products, 9 copies, 10 and 11 look over values. A block works on two things in turn, so that the tensor
// pipe runs one while the softmax warps are at the other:
//   two tiles (ONE = false)   A and B, 2 * (128 / G) consecutive tokens, sharing every key tile
//   one tile (ONE = true)     few rows: the even and the odd key tiles of the same queries, each with a softmax of its own; joined later
// Keys may be split further over `parts` blocks. Whatever is split leaves (maximum, sum, unnormalised output) in scratch for attn_paged_join_kernel.
//
// Pages: a tile of 128 keys is 128 / page boxes (or part of a page); the lanes of the copying warp look the pages up, well ahead. A page that
// the table does not name, or that begins behind the last position any row sees, is not fetched, and its keys are hidden by a bit mask.
// What lies at hidden positions must not count: scores are replaced by index, but a weight of zero times a value that is not finite is not zero, and
// places that were not fetched hold anything. So in tiles where some row does not see some key, two warps put zeros over values that no row sees, and over those
// that are not finite; if there were any of the latter (`poison`), the rows that do see them add them at the end.
#include <algorithm>

#include "attention_paged.cuh"

using namespace tc;

namespace {

constexpr int BQ = 128, BKV = 128;
constexpr int THREADS = 384;
constexpr float LOG2E = 1.4426950408889634f;

struct TilesArgs {
  PagedAttnArgs a;
  PagedJoin join;  // parts of the output: ONE: 2 * parts, otherwise parts
  int parts, ct;   // blocks that share the keys, tiles of a piece
  int G, tw;       // heads per key/value head, tokens of a tile of 128 rows
  double inv_tb;   // 1 / tokens of a block
  int* status;
};

// What a block works on, the same in all of its threads.
struct Work {
  int b, hk, part;
  int64_t row0;          // first row in q and out
  int n;                 // tokens
  int lo_pos;            // position of the first token
  int lo_key;            // first key in the window of the first token
  PagedWalk w;
  int nt;                // key tiles of this block
};

// What the issuing warp executes as a whole, one lane of it acting: operands that the compiler knows to be the same in all lanes need not be moved to
// uniform registers one by one in front of every instruction (a lane on its own took 85 to 120 cycles per product, more than the product).
__device__ __forceinline__ uint32_t elected() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < WAIT_LIMIT; i++) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
  }
  return false;
}
__device__ __forceinline__ void warp_mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void warp_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void warp_commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead)
      : "memory");
}

// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// key (and value) tiles in shared memory: what 227 KB hold beside the queries
template <int QA, bool ONE>
constexpr int tiles_ring() { return QA == 1 ? 4 : ONE ? 3 : 2; }
template <int QA, bool ONE>
constexpr size_t tiles_smem() { return (size_t)((ONE ? 1 : 2) + 2 * tiles_ring<QA, ONE>()) * QA * HALF_BYTES + 1024; }

// The x-th unit of work, a tile of tb tokens of a sequence, in the order of falling positions (of the last token, by 128): the blocks with the most keys
// start first, those of all sequences, and the short ones fill the SMs at the end. (Sequence by sequence, 4 prompts of 683 to 2048 tokens took 174 us
// instead of TIME_LPT.) Nobody lists the units: how many of them end at position X or later is a sum over the sequences, so the level of the x-th is searched
// for, and its sequence found in that level. False behind the last unit. A warp calls it together.
struct UnitSeq {
  int past, n, units;  // of sequence lane + 32 i: tokens before the new ones, new ones, tiles
};
__device__ __forceinline__ int units_from(const UnitSeq& u, int X, double inv_tb) {  // its units that end at X or later
  if (X <= 0) return u.units;
  if (u.past + u.n < X) return 0;
  return u.units - (X > u.past ? (int)((X - u.past - 1 + 0.5) * inv_tb) : 0);  // (X - past - 1) / tb units end before
}
__device__ bool find_unit(const PagedView& v, int tb, double inv_tb, int x, int lane, int* b_out, int* tile_out) {
  constexpr int KEEP = 4;  // sequences of a lane that stay in registers; more are read again each time
  auto seq = [&](int b) {
    UnitSeq u{0, 0, 0};
    if (b < v.B) {
      u.n = max(0, v.starts[b + 1] - v.starts[b]);
      u.past = v.lens[b] - u.n;
      u.units = (int)((u.n + tb - 1 + 0.5) * inv_tb);
    }
    return u;
  };
  UnitSeq kept[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; i++) kept[i] = seq(lane + 32 * i);
  int top = 0;
#pragma unroll
  for (int i = 0; i < KEEP; i++)
    if (kept[i].n) top = max(top, kept[i].past + kept[i].n);
  for (int b = lane + 32 * KEEP; b < v.B; b += 32) {
    const UnitSeq u = seq(b);
    if (u.n) top = max(top, u.past + u.n);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  auto from = [&](int X) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < KEEP; i++) c += units_from(kept[i], X, inv_tb);
    for (int b = lane + 32 * KEEP; b < v.B; b += 32) c += units_from(seq(b), X, inv_tb);
    return __reduce_add_sync(0xffffffffu, c);
  };
  if (x >= from(0)) return false;
  int lo = 0, hi = top / BKV + 1, below = 0;  // from(128 lo) > x >= from(128 hi) = below
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, c = from(mid * BKV);
    if (c > x) lo = mid;
    else hi = mid, below = c;
  }
  int rest = x - below;
  for (int b0 = 0; b0 < v.B; b0 += 32) {
    const UnitSeq u = seq(b0 + lane);
    const int first = u.units - units_from(u, lo * BKV, inv_tb), c = u.units - first - units_from(u, hi * BKV, inv_tb);
    int sum = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const unsigned there = __ballot_sync(0xffffffffu, sum > rest);
    if (there) {
      const int src = __ffs(there) - 1;
      *b_out = b0 + src;
      *tile_out = __shfl_sync(0xffffffffu, first + rest - (sum - c), src);
      return true;
    }
    rest -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

template <int QA, bool ONE>
__global__ void __launch_bounds__(THREADS) attn_paged_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TilesArgs t) {
  constexpr int TILE = QA * HALF_BYTES, NQ = ONE ? 1 : 2, D = 64 * QA, RING = tiles_ring<QA, ONE>();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t bar_q, k_full[RING], k_empty[RING], v_full[RING], v_ready[RING], v_empty[RING], bar_s[2], bar_p[2][2], bar_o[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ uint32_t page_bits[8];  // pages of a key tile that are there
  __shared__ int poison;
  const PagedAttnArgs& a = t.a;
  pdl_wait();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  Work k;
  {
    const int per = a.Hkv * t.parts;
    k.part = blockIdx.x % per / a.Hkv;
    k.hk = blockIdx.x % a.Hkv;
    int tile;
    if (!find_unit(a.at, NQ * t.tw, t.inv_tb, blockIdx.x / per, lane, &k.b, &tile)) return;
    const int sb = a.at.starts[k.b], n_new = a.at.starts[k.b + 1] - sb, len = a.at.lens[k.b], q0 = tile * NQ * t.tw;
    if (sb < 0 || (int64_t)sb + n_new > a.at.T || q0 < 0 || q0 >= n_new) return;  // starts or lengths that are none
    k.row0 = sb + q0;
    k.n = min(NQ * t.tw, n_new - q0);
    k.lo_pos = len - n_new + q0;
    k.lo_key = a.window ? max(0, k.lo_pos - a.window + 1) : 0;
    k.w = paged_walk(a.at, len, k.lo_pos, k.lo_pos + k.n - 1, a.window, a.first, BKV);
    k.nt = share_count(k.w.total, k.part, t.parts, t.ct);
  }
  // key tiles of each stream: ONE: every other one; otherwise tile A ends where its last token does
  int nt[2];
  if (ONE) {
    nt[0] = (k.nt + 1) / 2;
    nt[1] = k.nt / 2;
  } else {
    const int end_a = max(0, min(k.w.end, k.lo_pos + min(k.n, t.tw)));
    nt[0] = min(k.nt, share_count(k.w.first + max(0, (end_a + BKV - 1) / BKV - k.w.lo), k.part, t.parts, t.ct));
    nt[1] = k.n > t.tw ? k.nt : 0;
    k.nt = max(nt[0], nt[1]);
  }
  auto tile_key = [&](int i) { return k.w.tile(share_tile(i, k.part, t.parts, t.ct)) * BKV; };  // first key of the block's i-th tile

  const uint32_t sQ = smem_u32(smem), sK = sQ + NQ * TILE, sV = sK + RING * TILE;
  // The copying warp sets up the barriers, requests what has room and meets the others at the barrier below.
  const int box = min(a.at.page, BKV), boxes = BKV / box;  // keys of a box; boxes of a tile
  int ready = 0;  // key and value tiles requested
  auto page_of = [&](int i, int x) {
    const int j = i < k.nt ? tile_key(i) + x * box : k.w.end;
    return j < k.w.end ? paged_page(a.at, k.b, j >> a.at.shift) : -1;
  };
  PageNames names;
  unsigned there = 0;
  auto copy_box = [&](const CUtensorMap* map, uint32_t tile, int i, int page, uint32_t bar) {
    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(there) * box * 128 * QA));
    __syncwarp();
    if (page >= 0) {
      const int row = (int)((page * (int64_t)a.Hkv + k.hk) * a.at.page) + ((tile_key(i) + lane * box) & (a.at.page - 1));
      for (int x = 0; x < QA; x++) tma_load_2d(tile + x * HALF_BYTES + lane * box * 128, map, x * 64, row, bar);
    }
  };
  auto copy_k = [&](int i) {
    const int page = names.of(i, boxes, lane, page_of), st = i % RING;
    there = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0) page_bits[i & 7] = there;
    copy_box(&map_k, sK + st * TILE, i, page, smem_u32(&k_full[st]));
    return page;
  };
  auto copy_v = [&](int i, int page) { copy_box(&map_v, sV + i % RING * TILE, i, page, smem_u32(&v_full[i % RING])); };
  if (warp == 9) {
    if (lane == 0) {
      mbar_init(smem_u32(&bar_q), 1);
      for (int i = 0; i < RING; i++) {
        mbar_init(smem_u32(&k_full[i]), 1); mbar_init(smem_u32(&k_empty[i]), 1);
        mbar_init(smem_u32(&v_full[i]), 1); mbar_init(smem_u32(&v_ready[i]), 64); mbar_init(smem_u32(&v_empty[i]), 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(smem_u32(&bar_s[i]), 1); mbar_init(smem_u32(&bar_p[i][0]), BQ); mbar_init(smem_u32(&bar_p[i][1]), BQ); mbar_init(smem_u32(&bar_o[i]), 1);
      }
      poison = 0;
      asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (k.nt > 0) {
      names.begin(boxes, lane, page_of);
      if (lane == 0) {
        const uint32_t bytes = (uint32_t)(t.G * t.tw * 128 * QA);
        const int nq = !ONE && nt[1] ? 2 : 1;
        mbar_expect_tx(smem_u32(&bar_q), nq * bytes);
        for (int w = 0; w < nq; w++)
          for (int i = 0; i < QA; i++) tma_load_3d(sQ + w * TILE + i * HALF_BYTES, &map_q, i * 64, k.hk * t.G, (int)(k.row0 + w * t.tw), smem_u32(&bar_q));
      }
      __syncwarp();
      for (; ready < min(k.nt, RING); ready++) copy_v(ready, copy_k(ready));
    }
  }
  if (warp == 8) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = tmem_base_slot;
  constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  constexpr uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);

  if (warp == 9) {
    // ---- copies, the first of them requested already
    bool good = true;
    for (int i = ready; i < k.nt; i++) {
      const int st = i % RING;
      const uint32_t ph = (uint32_t)(i / RING & 1) ^ 1;
      good = warp_wait(smem_u32(&k_empty[st]), ph);
      if (!good) { if (lane == 0) set_status(t.status, 41); break; }
      const int page = copy_k(i);
      good = warp_wait(smem_u32(&v_empty[st]), ph);
      if (!good) { if (lane == 0) { set_status(t.status, 42); mbar_wait(smem_u32(&k_full[st]), ph ^ 1); } break; }
      copy_v(i, page);
      ready = i + 1;
    }
    // copies in flight have landed before this block's memory is somebody else's; only needed where the waits of the others gave up
    if (lane == 0 && k.nt > 0) {
      mbar_wait(smem_u32(&bar_q), 0);
      for (int i = max(0, ready - RING); i < ready; i++) {
        mbar_wait(smem_u32(&k_full[i % RING]), (uint32_t)(i / RING & 1));
        mbar_wait(smem_u32(&v_full[i % RING]), (uint32_t)(i / RING & 1));
      }
    }
    __syncwarp();
  } else if (warp == 8) {
    // ---- products
    const int n0 = __shfl_sync(0xffffffffu, nt[0], 0), n1 = __shfl_sync(0xffffffffu, nt[1], 0), n_all = __shfl_sync(0xffffffffu, k.nt, 0);
    if (n_all > 0) {
      const uint32_t lead = elected();
      auto issue_s = [&](int w, int st) {
        const uint32_t tS = tmem + (uint32_t)(w * 256);
#pragma unroll
        for (int s = 0; s < 4 * QA; s++) {
          const uint32_t off = (uint32_t)((s >> 2) * HALF_BYTES + (s & 3) * 32);
          warp_mma_ss(lead, tS, desc_kmajor(sQ + (ONE ? 0 : w * TILE) + off), desc_kmajor(sK + st * TILE + off), idesc_s, s ? 1u : 0u);
        }
        warp_commit(lead, smem_u32(&bar_s[w]));
      };
      auto issue_pv = [&](int w, int st, bool first, uint32_t ph) {  // by halves of the keys, as their weights come
        const uint32_t tS = tmem + (uint32_t)(w * 256), tO = tS + 128;
#pragma unroll
        for (int s = 0; s < 8; s++) {
          if ((s & 3) == 0) {
            if (!warp_wait(smem_u32(&bar_p[w][s >> 2]), ph)) return false;
            tc_fence_after();
          }
          const uint64_t dv = desc_mnmajor(sV + st * TILE + (uint32_t)(s * 2048));
          const uint32_t pcol = (uint32_t)((s >> 1) * 32 + (s & 1) * 8);
          warp_mma_ts(lead, tO, tS + pcol, dv, idesc_pv, (s || !first) ? 1u : 0u);
          warp_mma_ts(lead, tO, tS + pcol + 16, dv, idesc_pv, 1u);
        }
        warp_commit(lead, smem_u32(&bar_o[w]));
        return true;
      };
      bool good = warp_wait(smem_u32(&bar_q), 0);
      if (ONE) {
        for (int w = 0; w < 2 && good; w++) {
          if ((w ? n1 : n0) == 0) break;
          good = warp_wait(smem_u32(&k_full[w]), 0);
          if (!good) break;
          tc_fence_after();
          issue_s(w, w);
          warp_commit(lead, smem_u32(&k_empty[w]));
        }
        for (int s = 0; s < n0 && good; s++) {
          for (int w = 0; w < 2 && good; w++) {
            if (s >= (w ? n1 : n0)) break;
            const int i = 2 * s + w;
            good = warp_wait(smem_u32(&v_ready[i % RING]), (uint32_t)(i / RING & 1)) && issue_pv(w, i % RING, s == 0, (uint32_t)(s & 1));
            if (!good) break;
            warp_commit(lead, smem_u32(&v_empty[i % RING]));
            if (s + 1 < (w ? n1 : n0)) {
              const int in = i + 2;
              good = warp_wait(smem_u32(&k_full[in % RING]), (uint32_t)(in / RING & 1));
              if (!good) break;
              tc_fence_after();
              issue_s(w, in % RING);
              warp_commit(lead, smem_u32(&k_empty[in % RING]));
            }
          }
        }
      } else {
        good = good && warp_wait(smem_u32(&k_full[0]), 0);
        if (good) {
          tc_fence_after();
          for (int w = 0; w < 2; w++)
            if ((w ? n1 : n0) > 0) issue_s(w, 0);
          warp_commit(lead, smem_u32(&k_empty[0]));
        }
        for (int i = 0; i < n_all && good; i++) {
          const int st = i % RING, in = (i + 1) % RING;
          good = warp_wait(smem_u32(&v_ready[st]), (uint32_t)(i / RING & 1));
          bool k_next = false;
          for (int w = 0; w < 2 && good; w++) {
            if (i < (w ? n1 : n0)) {
              good = issue_pv(w, st, i == 0, (uint32_t)(i & 1));
              if (!good) break;
            }
            if (i + 1 < (w ? n1 : n0)) {
              if (!k_next) {
                good = warp_wait(smem_u32(&k_full[in]), (uint32_t)((i + 1) / RING & 1));
                if (!good) break;
                tc_fence_after();
                k_next = true;
              }
              issue_s(w, in);
            }
          }
          if (!good) break;
          warp_commit(lead, smem_u32(&v_empty[st]));
          if (i + 1 < n_all) warp_commit(lead, smem_u32(&k_empty[in]));
        }
      }
      if (!good) {  // what was issued has ended before the tiles are somebody else's
        if (lane == 0) set_status(t.status, 43);
        warp_commit(lead, smem_u32(&bar_q));
        warp_wait(smem_u32(&bar_q), 1);
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---- values of tiles that not every row sees whole
    const int tid = (int)threadIdx.x - 10 * 32;
    bool good = true;
    for (int i = 0; i < k.nt && good; i++) {
      const int st = i % RING, k0 = tile_key(i);
      good = mbar_wait(smem_u32(&v_full[st]), (uint32_t)(i / RING & 1));
      if (!good) break;
      const uint32_t bits = page_bits[i & 7];
      if (bits != (1u << boxes) - 1 || !sees_all(a, k.w.end, k0, BKV, k.lo_pos, k.lo_pos + k.n - 1)) {
        uint32_t found = 0;
        uint4* v = (uint4*)(smem + (NQ + RING + st) * TILE);
        for (int x = tid; x < QA * BKV * 8; x += 64) {
          const int r = (x >> 3) & (BKV - 1), j = k0 + r;
          const bool seen = j < k.w.end && (bits >> (r / box) & 1) && (j >= k.lo_key || j < a.first);
          if (!seen) {
            v[x] = make_uint4(0, 0, 0, 0);
            continue;
          }
          const uint4 w = v[x];
          if (not_finite(w.x) | not_finite(w.y) | not_finite(w.z) | not_finite(w.w)) {
            v[x] = make_uint4(only_finite(w.x), only_finite(w.y), only_finite(w.z), only_finite(w.w));
            found = 1;
          }
        }
        if (found) poison = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&v_ready[st])) : "memory");
    }
    if (!good && lane == 0) set_status(t.status, 44);
  } else {
    // ---- softmax of stream w, a thread per row: its 128 scores stay in registers between the maximum and the exponentials
    const int w = warp >> 2, row = (int)threadIdx.x & (BQ - 1);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + (uint32_t)(w * 256), tO = tS + 128;
    const int tok = row / t.G + (ONE ? 0 : w * t.tw);
    const bool live = row < t.G * t.tw && tok < k.n;
    const bool any_live = __any_sync(0xffffffffu, live);  // a warp without rows only keeps step
    const int pos_a = k.lo_pos + (ONE ? 0 : w * t.tw), pos_b = k.lo_pos + min(k.n, (ONE ? 1 : 1 + w) * t.tw) - 1;  // positions of the stream's tokens
    const int pos = k.lo_pos + tok;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0;
    const float scale_log2 = a.scale * LOG2E;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;  // after a wait that gave up the steps go on without waiting
    for (int s = 0; s < nt[w]; s++) {
      const uint32_t ph = (uint32_t)(s & 1);
      const int i = ONE ? 2 * s + w : s;
      ok = ok && mbar_wait(smem_u32(&bar_s[w]), ph);
      __syncwarp();  // the loads from tensor memory want the warp together
      tc_fence_after();
      if (any_live) {
        uint32_t r[BKV];
        tc_ld32(tS + lane_base, r);
        tc_ld32(tS + lane_base + 32, r + 32);
        const int k0 = tile_key(i);
        const uint32_t bits = page_bits[i & 7];
        const bool full = bits == (1u << boxes) - 1 && sees_all(a, k.w.end, k0, BKV, pos_a, pos_b);
        tc_wait_ld();
        tc_ld32(tS + lane_base + 64, r + 64);  // on their way while the maximum of the first half is taken
        tc_ld32(tS + lane_base + 96, r + 96);
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (full) {
#pragma unroll
          for (int j = 0; j < 64; j += 2) m4[(j >> 1) & 3] = max3(m4[(j >> 1) & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        }
        tc_wait_ld();
        if (!full) {
          // keys [0, hi) of the tile without [first, lo) and without pages that are not there
          const int hi = min(k.w.end, pos + 1) - k0, lw = lo - k0, fi = a.first - k0;
#pragma unroll
          for (int c = 0; c < 4; c++) {
            auto below = [&](int x) { return x - c * 32 >= 32 ? ~0u : x - c * 32 > 0 ? (1u << (x - c * 32)) - 1 : 0u; };
            uint32_t see = below(hi) & (~below(lw) | below(fi));
            if (!(bits >> (c * 32 / box) & 1)) see &= 0xFFFF0000u;
            if (!(bits >> ((c * 32 + 16) / box) & 1)) see &= 0x0000FFFFu;
#pragma unroll
            for (int j = 0; j < 32; j++)
              if (!(see >> j & 1)) r[c * 32 + j] = 0xFF800000u;  // -inf
          }
#pragma unroll
          for (int j = 0; j < 64; j += 2) m4[(j >> 1) & 3] = max3(m4[(j >> 1) & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        }
#pragma unroll
        for (int j = 64; j < BKV; j += 2) m4[(j >> 1) & 3] = max3(m4[(j >> 1) & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        const float m_tile = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale_log2;
        const bool grow = m_tile > m_run + 8.0f;
        const float m_use = grow ? m_tile : m_run;
        const float corr = grow ? exp2f(m_run - m_use) : 1.0f;
        m_run = m_use;
        const float base = m_use == -INFINITY ? 0.f : -m_use;
        if (s > 0 && __any_sync(0xffffffffu, grow)) {
          ok = ok && mbar_wait(smem_u32(&bar_o[w]), ph ^ 1);  // the product in front has finished O
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 4 * QA; c++) {
            uint32_t x[16];
            tc_ld16(tO + lane_base + (uint32_t)(c * 16), x);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * corr);
            tc_st16(tO + lane_base + (uint32_t)(c * 16), x);
          }
        }
        const uint64_t scale2 = pack2(__float_as_uint(scale_log2), __float_as_uint(scale_log2)), base2 = pack2(__float_as_uint(base), __float_as_uint(base));
        const uint64_t minus = pack2(0xBF800000u, 0xBF800000u);  // -1, -1
        uint64_t sum = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          uint32_t hi[16], lo16[16];
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const uint64_t e = fma2(pack2(r[c * 32 + 2 * j], r[c * 32 + 2 * j + 1]), scale2, base2);
            const uint32_t b0 = __float_as_uint(ex2_approx(__uint_as_float((uint32_t)e))), b1 = __float_as_uint(ex2_approx(__uint_as_float((uint32_t)(e >> 32))));
            const uint64_t p = pack2(b0, b1);
            sum = add2(sum, p);
            hi[j] = __byte_perm(b0, b1, 0x7632);
            const uint64_t rest = fma2(pack2(b0 & 0xFFFF0000u, b1 & 0xFFFF0000u), minus, p);
            lo16[j] = __byte_perm((uint32_t)rest, (uint32_t)(rest >> 32), 0x7632);
          }
          tc_st16(tS + lane_base + (uint32_t)(c * 32), hi);
          tc_st16(tS + lane_base + (uint32_t)(c * 32 + 16), lo16);
          if (c == 1) {  // the product of the first 64 keys may begin
            tc_wait_st();
            tc_fence_before();
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bar_p[w][0])) : "memory");
          }
        }
        l_run = l_run * corr + (__uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32)));
        tc_wait_st();
      } else {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bar_p[w][0])) : "memory");
      }
      tc_fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bar_p[w][1])) : "memory");
    }
    if (nt[w] > 0) {
      ok = ok && mbar_wait(smem_u32(&bar_o[w]), (uint32_t)((nt[w] - 1) & 1));
      __syncwarp();
      tc_fence_after();
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && lane == 0) set_status(t.status, 45);
    if (ok && any_live) {
      const int64_t at = (k.row0 + tok) * a.Hq + k.hk * t.G + row % t.G;
      const int np = ONE ? 2 * t.parts : t.parts, p = ONE ? 2 * k.part + w : k.part;
      const bool split = np > 1;
      const float inv = split ? 1.f : l_run == 0.f ? 0.f : 1.0f / l_run;
      if (split && live) t.join.ml[at * np + p] = make_float2(m_run, l_run);
      const bool bad = *(volatile int*)&poison;
      // Finished rows go through the queries' place in shared memory, which nobody reads any more, so that a warp's stores are whole rows (a thread per row
      // and store is 32 lines for 512 bytes: 4700 cycles of a block).
      uint4* stage = (uint4*)(smem + (ONE ? 0 : w * TILE)) + (row & ~31) * (D / 8);  // 32 rows of this warp, chunk c of row r at c ^ (r & 7)
      if (!split && nt[w] == 0 && k.nt > 0) mbar_wait(smem_u32(&bar_q), 0);  // the queries have come there
#pragma unroll 1
      for (int c = 0; c < 2 * QA; c++) {
        uint32_t r[32];
        __syncwarp();
        if (nt[w] > 0) {
          tc_ld32(tO + lane_base + (uint32_t)(c * 32), r);
          tc_wait_ld();
        }
        if (l_run == 0.f) {
#pragma unroll
          for (int j = 0; j < 32; j++) r[j] = 0;
        } else if (bad && live) {
          float f[32];
          for (int j = 0; j < 32; j++) f[j] = __uint_as_float(r[j]);
          add_poison(a, k.w, k.b, k.hk, k.part, t.parts, t.ct, BKV, ONE ? w : 0, ONE ? 2 : 1, nt[w], pos, c * 32, 32, f);
          for (int j = 0; j < 32; j++) r[j] = __float_as_uint(f[j]);
        }
        if (split) {
          if (live && l_run != 0.f) {
            float* dst = t.join.o + (at * np + p) * D + c * 32;
#pragma unroll
            for (int j = 0; j < 32; j += 4) *(uint4*)(dst + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 v;
            v.x = f32_to_bf16_bits(__uint_as_float(r[j]) * inv) | (f32_to_bf16_bits(__uint_as_float(r[j + 1]) * inv) << 16);
            v.y = f32_to_bf16_bits(__uint_as_float(r[j + 2]) * inv) | (f32_to_bf16_bits(__uint_as_float(r[j + 3]) * inv) << 16);
            v.z = f32_to_bf16_bits(__uint_as_float(r[j + 4]) * inv) | (f32_to_bf16_bits(__uint_as_float(r[j + 5]) * inv) << 16);
            v.w = f32_to_bf16_bits(__uint_as_float(r[j + 6]) * inv) | (f32_to_bf16_bits(__uint_as_float(r[j + 7]) * inv) << 16);
            stage[lane * (D / 8) + ((c * 4 + j / 8) ^ (lane & 7))] = v;
          }
        }
      }
      if (!split) {
        __syncwarp();
        constexpr int LANES = D / 8, PASS = 32 / LANES;  // lanes of a row, rows of a pass
#pragma unroll 4
        for (int x = 0; x < 32; x += PASS) {
          const int rr = x + lane / LANES, cc = lane % LANES;
          const int64_t to = __shfl_sync(0xffffffffu, at, rr);
          const bool on = __shfl_sync(0xffffffffu, (int)live, rr);
          const uint4 v = stage[rr * LANES + (cc ^ (rr & 7))];
          if (on) *(uint4*)(a.out + to * D + cc * 8) = v;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// [T, heads, cols], boxes of `tokens` x G heads x 64 columns
int map_tokens(CUtensorMap* map, const void* base, int64_t T, int heads, int cols, int G, int tokens) {
  EncodeFn encode;
  SB_TRY(encode_fn(&encode));
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)heads, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * heads * 2};
  cuuint32_t boxes[3] = {64u, (cuuint32_t)G, (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sb_fail(STRICTB200_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return STRICTB200_OK;
}

template <int QA, bool ONE>
int launch(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  TilesArgs t;
  t.a = a;
  t.G = a.Hq / a.Hkv;
  t.tw = BQ / t.G;
  t.status = ctx->d_status;
  const int tb = (ONE ? 1 : 2) * t.tw;
  t.inv_tb = 1.0 / tb;
  const int64_t tiles = a.at.T / tb + a.at.B;  // room for the tiles of all sequences
  // Parts: the fewest rounds of key tiles over the SMs, a block counted with three tiles more (its start and its end) and the join with four.
  const int64_t units = std::max<int64_t>((a.at.T + tb - 1) / tb, a.at.B) * a.Hkv, keys = std::max<int64_t>(1, paged_walk_tiles(a, BKV));
  int64_t best = INT64_MAX;
  t.parts = 1;
  for (int p = 1; p <= 64 && p <= keys; p++) {
    if (p > 1 && (size_t)a.at.T * a.Hq * p * (ONE ? 2 : 1) * (64 * QA + 2) * 4 > ((size_t)256 << 20)) break;
    const int64_t cost = (units * p + ctx->sm_count - 1) / ctx->sm_count * ((keys + p - 1) / p + 3) + (p > 1 ? 4 : 0);
    if (cost < best) best = cost, t.parts = p;
  }
  t.ct = (int)((keys + t.parts - 1) / t.parts);
  const int np = (ONE ? 2 : 1) * t.parts;
  if (np > 1) SB_TRY(paged_join_scratch(ctx, a, np, &t.join));
  const int64_t blocks = tiles * a.Hkv * t.parts;
  if (blocks > INT32_MAX) return sb_fail(STRICTB200_ERR_UNSUPPORTED, "attention: too many rows and heads for one call");
  CUtensorMap mq, mk, mv;
  const int64_t rows = (int64_t)a.at.n_pages * a.Hkv * a.at.page;
  SB_TRY(map_tokens(&mq, a.q, a.at.T, a.Hq, a.D, t.G, t.tw));
  SB_TRY(paged_map_rows(&mk, a.k, rows, a.D, std::min(a.at.page, BKV)));
  SB_TRY(paged_map_rows(&mv, a.v, rows, a.D, std::min(a.at.page, BKV)));
  constexpr size_t smem = tiles_smem<QA, ONE>();
  static SbDeviceOnce once;  // one per instantiation
  SB_CUDA(once.run(ctx->device, [&] { return cudaFuncSetAttribute(attn_paged_tiles_kernel<QA, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
  SB_CUDA(sb_launch(ctx, attn_paged_tiles_kernel<QA, ONE>, dim3((unsigned)blocks), dim3(THREADS), smem, mq, mk, mv, t));
  ctx->launches++;
  return np > 1 ? paged_join(ctx, a, t.join) : STRICTB200_OK;
}

}  // namespace

int k_attn_paged_tiles(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  const bool one = (int64_t)a.max_new * (a.Hq / a.Hkv) <= BQ;  // one tile per sequence
  if (a.D == 128) return one ? launch<2, true>(ctx, a) : launch<2, false>(ctx, a);
  return one ? launch<1, true>(ctx, a) : launch<1, false>(ctx, a);
}
