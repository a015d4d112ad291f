// Softmax attention of new tokens over a paged cache on the tcgen05 tensor cores: drafted tokens, chunks and whole prompts.
//
// A row of the products is one query head of one new token: the G heads that share a key/value head are packed behind one another, 128 / G tokens to a
// tile of 128 rows (one TMA box: 64 dims x G heads x tokens), so keys and values are fetched once for all of them and a tile spans few positions. Rows
// are lanes of tensor memory. Per tile of 128 keys, as in the attention over contiguous caches:
//   S = Q K^T      operands in shared memory, fp32 sums in tensor memory
//   softmax        a thread per row, running maximum followed lazily (a row of O is rescaled when its maximum grew by more than 2^8), weights back to
//                  tensor memory as two bf16 terms (hi + lo by truncation: 2^-16)
//   O += P V       weights from tensor memory, values from shared memory; O stays in tensor memory
// Blocks stay (one per SM) and take one unit after the other: a tile of tokens, a key/value head and a share of the keys. Roles: warps 0..7 softmax, 8 issues
// products, 9 finds units, announces them (two ahead of the slowest) and copies, 10 and 11 look over values. They meet at mbarriers only, so the copies and
// first products of a unit run while the last one's rows are being written. (A block per unit cost 13 us a unit beside 2.5 us a key tile; now 4 to 7. 4 x 8192 tokens, 32 heads
// of 128: 2530 us, 868 TFLOP/s, of which three halves are executed; 4 x 2048 206 us.) A block
// works on two things in turn, so that the tensor pipe runs one while the softmax warps are at the other:
//   two tiles (ONE = false)   A and B, 2 * (128 / G) consecutive tokens, sharing every key tile
//   one tile (ONE = true)     few rows: the even and the odd key tiles of the same queries, each with a softmax of its own; joined later
// Keys may be split further over `parts` blocks. Whatever is split leaves (maximum, sum, unnormalised output) in scratch for attn_paged_join_kernel.
//
// Pages: a tile of 128 keys is 128 / page boxes (or part of a page); the lanes of the copying warp look the pages up, well ahead. A page that
// the table does not name, or that begins behind the last position any row sees, is not fetched, and its keys are hidden by a bit mask.
// What lies at hidden positions must not count: scores are replaced by index, but a weight of zero times a value that is not finite is not zero, and
// places that were not fetched hold anything. So in tiles where some row does not see some key, two warps put zeros over values that are not finite; if any
// row sees one of those (`poison`), it adds them at the end.
#include <algorithm>
#include <cmath>

#include "attention_paged.cuh"

using namespace tc;

namespace {

constexpr int BQ = 128, BKV = 128;
constexpr int THREADS = 384;
constexpr float LOG2E = 1.4426950408889634f;

struct TilesArgs {
  PagedAttnArgs a;
  PagedJoin join;  // parts of the output: ONE: 2 * parts, otherwise parts
  int parts;       // blocks that share the keys of a unit
  int G, tw;       // heads per key/value head, tokens of a tile of 128 rows
  double inv_tb;   // 1 / tokens of a unit
  int one_round;   // a block for every unit
  int direct;      // unit x is sequence x
  int* status;
};

// What a block works on.
struct Unit {
  int b, hk, part;
  int n;       // tokens; -1: there is no further unit
  int lo_pos;  // position of the first token
  int lo_key;  // first key in the window of the first token
  int64_t row0;  // first row in q and out
  PagedWalk w;
  int ct;           // tiles of a part: what a unit sees is cut evenly (pieces cut by the longest sequence took 132 us where these take 84, uneven drafts)
  int nt, nt_w[2];  // key tiles of the unit and of each stream
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
constexpr size_t tiles_smem() { return (size_t)((ONE ? 1 : 2) + 2 * tiles_ring<QA, ONE>()) * QA * HALF_BYTES + (ONE ? 0 : 8 * 4096) + 1024; }

// The x-th unit of work, a tile of tb tokens of a sequence, in the order of falling positions (of the last token, by 128): those with the most keys come
// first, of all sequences, and the short ones fill the SMs at the end. Nobody lists the units: how many of them end at position X or later is a sum over
// the sequences, so the level of the x-th is searched for, and its sequence found in that level. False behind the last unit. A warp calls it together.
// Where every unit has a block of its own the order does not matter: then the tiles of sequence b begin at (starts[b] - starts[0]) / tb + b, room for all.
__device__ __forceinline__ bool place_unit(const PagedView& v, double inv_tb, int x, int lane, int* b_out, int* tile_out) {
  const int s0 = v.starts[0];
  int before = 0, base = 0;
  for (int b0 = 0; b0 < v.B; b0 += 32) {
    const int b = b0 + lane, at = b < v.B ? (int)((v.starts[b] - s0 + 0.5) * inv_tb) + b : INT_MAX;
    const unsigned m = __ballot_sync(0xffffffffu, at <= x);
    if (m) base = __shfl_sync(0xffffffffu, at, 31 - __clz(m));
    before += __popc(m);
    if (m != 0xffffffffu) break;
  }
  *b_out = before - 1;
  *tile_out = x - base;
  return before > 0;
}
struct UnitSeq {
  int past, n, units;  // of sequence lane + 32 i: tokens before the new ones, new ones, tiles
};
__device__ __forceinline__ int units_from(const UnitSeq& u, int X, double inv_tb) {  // its units that end at X or later
  if (X <= 0) return u.units;
  if (u.past + u.n < X) return 0;
  return u.units - (X > u.past ? (int)((X - u.past - 1 + 0.5) * inv_tb) : 0);  // (X - past - 1) / tb units end before
}
// KEEP: sequences of a lane that stay in registers; more are read again each time.
template <int KEEP>
__device__ bool find_unit(const PagedView& v, int tb, double inv_tb, int x, int lane, int* b_out, int* tile_out) {
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
    const int first = u.units - units_from(u, lo * BKV, inv_tb), c = u.units - first - (hi > top / BKV ? 0 : units_from(u, hi * BKV, inv_tb));  // no unit ends there, and 128 hi may be 2^31
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

// Of a row of a unit: 32 dims from d0 on. Everything else is looked up again here (as arguments they cost the softmax warps registers: 185 us a chunk instead of 177).
__device__ __noinline__ void add_poison(const TilesArgs& t, const Unit& k, const Poison& noted, bool one, int w, int nt, int pos, int d0, float* r) {
  add_poison(t.a, k.w, k.b, k.hk, k.part, t.parts, k.ct, BKV, BKV, k.lo_pos, k.lo_pos + k.n - 1, noted, one ? w : 0, one ? 2 : 1, nt, pos, d0, 32, r);
}

template <int QA, bool ONE>
__global__ void __launch_bounds__(THREADS, 1) attn_paged_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                                                                   const __grid_constant__ TilesArgs t) {
  constexpr int TILE = QA * HALF_BYTES, NQ = ONE ? 1 : 2, D = 64 * QA, RING = tiles_ring<QA, ONE>();
  constexpr int READERS = 11;  // warps that read a unit's description
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t unit_full[2], unit_empty[2], q_full, q_empty, k_full[RING], k_empty[RING], v_full[RING], v_ready[RING], v_empty[RING], bar_s[2],
      bar_p[2][2], bar_o[2], o_free[2];
  __shared__ Unit units[2];
  __shared__ Poison poison[2];  // of these units
  __shared__ uint32_t tmem_base_slot;
  __shared__ uint32_t page_bits[8];  // pages of a key tile that are there
  const PagedAttnArgs& a = t.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t sQ = smem_u32(smem), sK = sQ + NQ * TILE, sV = sK + RING * TILE;
  if (warp == 9 && lane == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&unit_full[i]), 1); mbar_init(smem_u32(&unit_empty[i]), READERS);
      mbar_init(smem_u32(&bar_s[i]), 1); mbar_init(smem_u32(&bar_p[i][0]), BQ); mbar_init(smem_u32(&bar_p[i][1]), BQ); mbar_init(smem_u32(&bar_o[i]), 1);
      mbar_init(smem_u32(&o_free[i]), BQ);
    }
    mbar_init(smem_u32(&q_full), 1); mbar_init(smem_u32(&q_empty), 1);
    for (int i = 0; i < RING; i++) {
      mbar_init(smem_u32(&k_full[i]), 1); mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&v_full[i]), 1); mbar_init(smem_u32(&v_ready[i]), 64); mbar_init(smem_u32(&v_empty[i]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  if (warp == 8) {
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
  const int box = min(a.at.page, BKV), boxes = BKV / box;  // keys of a box; boxes of a tile
  // A count of phases over all units gives each wait its parity. next_unit: the description of the u-th unit, false behind the last or after a wait that gave up.
  auto next_unit = [&](int u) { return warp_wait(smem_u32(&unit_full[u & 1]), (uint32_t)(u >> 1 & 1)) && units[u & 1].n >= 0; };
  auto unit_read = [&](int u) {
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&unit_empty[u & 1])) : "memory");
  };

  // Registers: 384 threads begin with 168 each; the softmax warps end up with 216, the others with 72 (256 * 216 + 128 * 72 = 384 * 168).
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {
      // ---- units and copies
      int c = 0, nq = 0;  // key tiles, units with keys
      bool good = true;
      for (int u = 0; good; u++) {
        // every other round of the blocks goes backwards: who had the longest of one has the shortest of the next
        const int64_t y = (int64_t)u * gridDim.x + (u & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        const int per = a.Hkv * t.parts;
        Unit k;
        k.n = -1;
        k.nt = 0;
        int tile;
        const int x = (int)(y / per);
        const bool one_round = t.one_round;
        if (t.direct) k.b = x, tile = 0;
        if (t.direct ? x < a.at.B : one_round ? u == 0 && place_unit(a.at, t.inv_tb, x, lane, &k.b, &tile)
                      : a.at.B <= 32 ? find_unit<1>(a.at, NQ * t.tw, t.inv_tb, x, lane, &k.b, &tile) : find_unit<4>(a.at, NQ * t.tw, t.inv_tb, x, lane, &k.b, &tile)) {
          k.part = (int)(y % per) / a.Hkv;
          k.hk = (int)(y % per) % a.Hkv;
          const int sb = a.at.starts[k.b], n_new = a.at.starts[k.b + 1] - sb, len = a.at.lens[k.b], q0 = tile * NQ * t.tw;
          k.row0 = (int64_t)sb + q0;
          k.lo_pos = len - n_new + q0;
          k.lo_key = window_begin(k.lo_pos, a.window);
          k.n = sb < 0 || (int64_t)sb + n_new > a.at.T || q0 < 0 ? 0 : max(0, min(NQ * t.tw, n_new - q0));  // nothing where starts or lengths are none
          k.w = paged_walk(a.at, len, k.lo_key, k.lo_pos + k.n - 1, a.first, BKV);
          k.ct = max(1, (k.w.total + t.parts - 1) / t.parts);
          k.nt = k.n ? share_count(k.w.total, k.part, t.parts, k.ct) : 0;
          if (ONE) {  // every other tile
            k.nt_w[0] = (k.nt + 1) / 2;
            k.nt_w[1] = k.nt / 2;
          } else {    // tile A ends where its last token does
            const int end_a = max(0, min(k.w.end, k.lo_pos + min(k.n, t.tw)));
            k.nt_w[0] = min(k.nt, share_count(k.w.first + max(0, (end_a + BKV - 1) / BKV - k.w.lo), k.part, t.parts, k.ct));
            k.nt_w[1] = k.n > t.tw ? k.nt : 0;
            k.nt = max(k.nt_w[0], k.nt_w[1]);
          }
        }
        if (u >= 2) good = warp_wait(smem_u32(&unit_empty[u & 1]), (uint32_t)(u >> 1 & 1) ^ 1);
        if (!good) break;
        if (lane == 0) {
          units[u & 1] = k;
          poison[u & 1].n = 0;
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&unit_full[u & 1])) : "memory");
        }
        __syncwarp();
        if (k.n < 0) break;
        if (k.nt == 0) continue;
        auto tile_key = [&](int i) { return k.w.tile(share_tile(i, k.part, t.parts, k.ct)) * BKV; };
        auto page_of = [&](int i, int x) {
          const int j = i < k.nt ? tile_key(i) + x * box : k.w.end;
          return j < k.w.end ? paged_page(a.at, k.b, j >> a.at.shift) : -1;
        };
        auto copy_boxes = [&](const CUtensorMap* map, uint32_t tile, int row, unsigned there, uint32_t bar) {
          if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(there) * box * 128 * QA));
          __syncwarp();
          if (row >= 0)
            for (int x = 0; x < QA; x++) tma_load_2d(tile + x * HALF_BYTES + lane * box * 128, map, x * 64, row, bar);
        };
        PageNames names;
        names.begin(boxes, lane, page_of);
        for (int i = 0; i < k.nt; i++, c++) {
          const int st = c % RING, page = names.of(i, boxes, lane, page_of);
          const uint32_t ph = (uint32_t)(c / RING & 1) ^ 1;
          const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
          const int row = page < 0 ? -1 : (int)((page * (int64_t)a.Hkv + k.hk) * a.at.page) + ((tile_key(i) + lane * box) & (a.at.page - 1));
          if (c >= RING) good = warp_wait(smem_u32(&k_empty[st]), ph);
          if (!good) break;
          if (lane == 0) page_bits[c & 7] = there;
          copy_boxes(&map_k, sK + st * TILE, row, there, smem_u32(&k_full[st]));
          if (i == 0) {
            if (nq) good = warp_wait(smem_u32(&q_empty), (uint32_t)(nq & 1) ^ 1);
            if (good && lane == 0) {
              const int tiles = !ONE && k.nt_w[1] ? 2 : 1;
              mbar_expect_tx(smem_u32(&q_full), (uint32_t)(tiles * t.G * t.tw * 128 * QA));
              for (int w = 0; w < tiles; w++)
                for (int x = 0; x < QA; x++) tma_load_3d(sQ + w * TILE + x * HALF_BYTES, &map_q, x * 64, k.hk * t.G, (int)(k.row0 + w * t.tw), smem_u32(&q_full));
            }
            if (good) nq++;
          }
          if (good && c >= RING) good = warp_wait(smem_u32(&v_empty[st]), ph);
          if (!good) {
            warp_wait(smem_u32(&k_full[st]), ph ^ 1);  // landed before this block's memory is somebody else's
            break;
          }
          copy_boxes(&map_v, sV + st * TILE, row, there, smem_u32(&v_full[st]));
        }
      }
      if (!good && lane == 0) set_status(t.status, 41);
      // copies in flight have landed before this block's memory is somebody else's; only needed where the waits of the others gave up
      if (nq) warp_wait(smem_u32(&q_full), (uint32_t)(nq & 1) ^ 1);
      for (int i = max(0, c - RING); i < c; i++) {
        warp_wait(smem_u32(&k_full[i % RING]), (uint32_t)(i / RING & 1));
        warp_wait(smem_u32(&v_full[i % RING]), (uint32_t)(i / RING & 1));
      }
    } else if (warp == 8) {
      // ---- products
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
      int c = 0, nq = 0, step0 = 0, step1 = 0, used0 = 0, used1 = 0;  // key tiles, units with keys; steps and units of each stream
      bool good = true;
      for (int u = 0; good && next_unit(u); u++) {
        const int n_all = __shfl_sync(0xffffffffu, units[u & 1].nt, 0), n0 = __shfl_sync(0xffffffffu, units[u & 1].nt_w[0], 0),
                  n1 = __shfl_sync(0xffffffffu, units[u & 1].nt_w[1], 0);
        unit_read(u);
        if (n_all == 0) continue;
        // O of a stream belongs to the last unit until its rows have been read
        auto o_mine = [&](int w) { return (w ? used1 : used0) == 0 || warp_wait(smem_u32(&o_free[w]), (uint32_t)((w ? used1 : used0) & 1) ^ 1); };
        auto k_there = [&](int i) {
          const bool ok = warp_wait(smem_u32(&k_full[(c + i) % RING]), (uint32_t)((c + i) / RING & 1));
          tc_fence_after();
          return ok;
        };
        good = warp_wait(smem_u32(&q_full), (uint32_t)(nq & 1));
        if (ONE) {
          for (int w = 0; w < 2 && good; w++) {
            if ((w ? n1 : n0) == 0) break;
            good = k_there(w);
            if (!good) break;
            issue_s(w, (c + w) % RING);
            warp_commit(lead, smem_u32(&k_empty[(c + w) % RING]));
            if (w == n_all - 1) warp_commit(lead, smem_u32(&q_empty));
          }
          for (int s = 0; s < n0 && good; s++) {
            for (int w = 0; w < 2 && good; w++) {
              if (s >= (w ? n1 : n0)) break;
              const int i = 2 * s + w, st = (c + i) % RING;
              good = warp_wait(smem_u32(&v_ready[st]), (uint32_t)((c + i) / RING & 1)) && (s || o_mine(w)) &&
                     issue_pv(w, st, s == 0, (uint32_t)((w ? step1 : step0) + s & 1));
              if (!good) break;
              warp_commit(lead, smem_u32(&v_empty[st]));
              if (s + 1 < (w ? n1 : n0)) {
                good = k_there(i + 2);
                if (!good) break;
                issue_s(w, (c + i + 2) % RING);
                warp_commit(lead, smem_u32(&k_empty[(c + i + 2) % RING]));
                if (i + 2 == n_all - 1) warp_commit(lead, smem_u32(&q_empty));
              }
            }
          }
        } else {
          good = good && k_there(0);
          if (good) {
            for (int w = 0; w < 2; w++)
              if ((w ? n1 : n0) > 0) issue_s(w, c % RING);
            warp_commit(lead, smem_u32(&k_empty[c % RING]));
            if (n_all == 1) warp_commit(lead, smem_u32(&q_empty));
          }
          for (int i = 0; i < n_all && good; i++) {
            const int st = (c + i) % RING, in = (c + i + 1) % RING;
            good = warp_wait(smem_u32(&v_ready[st]), (uint32_t)((c + i) / RING & 1));
            bool k_next = false;
            for (int w = 0; w < 2 && good; w++) {
              if (i < (w ? n1 : n0)) {
                good = (i || o_mine(w)) && issue_pv(w, st, i == 0, (uint32_t)((w ? step1 : step0) + i & 1));
                if (!good) break;
              }
              if (i + 1 < (w ? n1 : n0)) {
                if (!k_next) {
                  good = k_there(i + 1);
                  if (!good) break;
                  k_next = true;
                }
                issue_s(w, in);
              }
            }
            if (!good) break;
            warp_commit(lead, smem_u32(&v_empty[st]));
            if (i + 1 < n_all) warp_commit(lead, smem_u32(&k_empty[in]));
            if (i + 2 == n_all) warp_commit(lead, smem_u32(&q_empty));
          }
        }
        c += n_all;
        nq++;
        step0 += n0;
        step1 += n1;
        used0 += n0 > 0;
        used1 += n1 > 0;
      }
      if (!good) {  // what was issued has ended before the tiles are somebody else's
        if (lane == 0) set_status(t.status, 43);
        warp_commit(lead, smem_u32(&k_empty[0]));
        for (int i = 0; i < 2; i++) warp_wait(smem_u32(&k_empty[0]), (uint32_t)i);
      }
    } else {
      // ---- values of tiles that not every row sees whole
      const int tid = (int)threadIdx.x - 10 * 32;
      int c = 0;
      bool good = true;
      for (int u = 0; good && next_unit(u); u++) {
        const Unit& k = units[u & 1];
        const PagedWalk w = k.w;
        const int nt = k.nt, part = k.part, ct = k.ct, lo_pos = k.lo_pos, hi_pos = k.lo_pos + k.n - 1, lo_key = k.lo_key;
        for (int i = 0; i < nt; i++, c++) {
          const int st = c % RING, k0 = w.tile(share_tile(i, part, t.parts, ct)) * BKV;
          good = warp_wait(smem_u32(&v_full[st]), (uint32_t)(c / RING & 1));
          if (!good) break;
          const uint32_t bits = page_bits[c & 7];
          if (bits != (1u << boxes) - 1 || !sees_all(a, w.end, k0, BKV, lo_pos, hi_pos)) {
            uint32_t found = 0;
            uint4* v = (uint4*)(smem + (NQ + RING + st) * TILE);
            constexpr int AHEAD = 8;  // finite values need nothing, whoever sees them: the loads of eight go together
            for (int x0 = tid; x0 < QA * BKV * 8; x0 += 64 * AHEAD) {
              uint4 y[AHEAD];
              uint32_t odd = 0;
#pragma unroll
              for (int e = 0; e < AHEAD; e++) y[e] = v[x0 + 64 * e];
#pragma unroll
              for (int e = 0; e < AHEAD; e++) odd |= not_finite(y[e].x) | not_finite(y[e].y) | not_finite(y[e].z) | not_finite(y[e].w);
              if (!odd) continue;
              for (int x = x0; x < x0 + 64 * AHEAD; x += 64) {
                const int r = (x >> 3) & (BKV - 1), j = k0 + r;
                const bool seen = j < w.end && (bits >> (r / box) & 1) && (j >= lo_key || j < a.first);
                const uint4 z = v[x];
                found |= seen && (not_finite(z.x) | not_finite(z.y) | not_finite(z.z) | not_finite(z.w));
                v[x] = make_uint4(only_finite(z.x), only_finite(z.y), only_finite(z.z), only_finite(z.w));
              }
            }
            if (__any_sync(0xffffffffu, found != 0) && lane == 0) note_poison(poison[u & 1], i);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&v_ready[st])) : "memory");
        }
        unit_read(u);
      }
      if (!good && lane == 0) set_status(t.status, 44);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax of stream w, a thread per row: its 128 scores stay in registers between the maximum and the exponentials
    const int w = warp >> 2, row = (int)threadIdx.x & (BQ - 1);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + (uint32_t)(w * 256), tO = tS + 128;
    const int tok = row / t.G + (ONE ? 0 : w * t.tw), head = row % t.G;
    const float scale_log2 = a.scale * LOG2E;
    int c = 0, steps = 0;  // key tiles of all units so far, steps of this stream
    bool good = true;
    for (int u = 0; good && next_unit(u); u++) {
      const Unit& k = units[u & 1];
      const int nt = k.nt_w[w], n_all = k.nt, part = k.part, ct = k.ct;
      const PagedWalk walk = k.w;
      const bool live = row < t.G * t.tw && tok < k.n;
      const bool any_live = __any_sync(0xffffffffu, live);  // a warp without rows only keeps step
      const int pos_a = k.lo_pos + (ONE ? 0 : w * t.tw), pos_b = k.lo_pos + min(k.n, (ONE ? 1 : 1 + w) * t.tw) - 1;  // positions of the stream's tokens
      const int pos = k.lo_pos + tok;
      const int lo = a.window ? max(0, (int)((uint32_t)pos - a.window + 1)) : 0;  // a row in front of its sequence sees nothing, wherever this lies
      float m_run = -INFINITY, l_run = 0.f;
      for (int s = 0; s < nt; s++, steps++) {
        const uint32_t ph = (uint32_t)(steps & 1);
        const int i = ONE ? 2 * s + w : s;
        good = warp_wait(smem_u32(&bar_s[w]), ph);
        if (!good) break;
        tc_fence_after();
        if (any_live) {
          uint32_t r[BKV];
          tc_ld32(tS + lane_base, r);
          tc_ld32(tS + lane_base + 32, r + 32);
          const int k0 = walk.tile(share_tile(i, part, t.parts, ct)) * BKV;
          const uint32_t bits = page_bits[(c + i) & 7];
          const bool full = bits == (1u << boxes) - 1 && sees_all(a, walk.end, k0, BKV, pos_a, pos_b);
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
            const int hi = min(walk.end, pos + 1) - k0, lw = lo - k0, fi = a.first - k0;
#pragma unroll
            for (int c4 = 0; c4 < 4; c4++) {
              auto below = [&](int x) { return x - c4 * 32 >= 32 ? ~0u : x - c4 * 32 > 0 ? (1u << (x - c4 * 32)) - 1 : 0u; };
              uint32_t see = below(hi) & (~below(lw) | below(fi));
              if (!(bits >> (c4 * 32 / box) & 1)) see &= 0xFFFF0000u;
              if (!(bits >> ((c4 * 32 + 16) / box) & 1)) see &= 0x0000FFFFu;
              if (__all_sync(0xffffffffu, see == ~0u)) continue;  // the rows of a warp are few tokens: most chunks are seen or hidden as a whole
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (!(see >> j & 1)) r[c4 * 32 + j] = 0xFF800000u;  // -inf
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
            good = warp_wait(smem_u32(&bar_o[w]), ph ^ 1);  // the product in front has finished O
            if (!good) break;
            tc_fence_after();
#pragma unroll 1
            for (int x16 = 0; x16 < 4 * QA; x16++) {
              uint32_t x[16];
              tc_ld16(tO + lane_base + (uint32_t)(x16 * 16), x);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * corr);
              tc_st16(tO + lane_base + (uint32_t)(x16 * 16), x);
            }
          }
          const uint64_t scale2 = pack2(__float_as_uint(scale_log2), __float_as_uint(scale_log2)), base2 = pack2(__float_as_uint(base), __float_as_uint(base));
          const uint64_t minus = pack2(0xBF800000u, 0xBF800000u);  // -1, -1
          uint64_t sum = 0;
#pragma unroll
          for (int c4 = 0; c4 < 4; c4++) {
            uint32_t hi[16], lo16[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
              const uint64_t e = fma2(pack2(r[c4 * 32 + 2 * j], r[c4 * 32 + 2 * j + 1]), scale2, base2);
              const uint32_t b0 = __float_as_uint(ex2_approx(__uint_as_float((uint32_t)e))), b1 = __float_as_uint(ex2_approx(__uint_as_float((uint32_t)(e >> 32))));
              const uint64_t p = pack2(b0, b1);
              sum = add2(sum, p);
              hi[j] = __byte_perm(b0, b1, 0x7632);
              const uint64_t rest = fma2(pack2(b0 & 0xFFFF0000u, b1 & 0xFFFF0000u), minus, p);
              lo16[j] = __byte_perm((uint32_t)rest, (uint32_t)(rest >> 32), 0x7632);
            }
            tc_st16(tS + lane_base + (uint32_t)(c4 * 32), hi);
            tc_st16(tS + lane_base + (uint32_t)(c4 * 32 + 16), lo16);
            if (c4 == 1) {  // the product of the first 64 keys may begin
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
      if (!good) break;
      if (nt > 0) {
        good = warp_wait(smem_u32(&bar_o[w]), (uint32_t)(steps & 1) ^ 1);
        if (!good) break;
        tc_fence_after();
      }
      const int64_t at = (k.row0 + tok) * a.Hq + k.hk * t.G + head;
      const int np = ONE ? 2 * t.parts : t.parts, p = ONE ? 2 * part + w : part;
      const float inv = np > 1 ? 1.f : l_run == 0.f ? 0.f : 1.0f / l_run;
      if (np > 1 && live) t.join.ml[at * np + p] = make_float2(m_run, l_run);
      const bool bad = __any_sync(0xffffffffu, *(volatile int*)&poison[u & 1].n > 0) && nt > 0 && any_live;  // of the warp; later tiles of the other stream may still add to it
      if (bad) {
#pragma unroll 1
        for (int c32 = 0; c32 < 2 * QA; c32++) {
          uint32_t r[32];
          float f[32];
          __syncwarp();
          tc_ld32(tO + lane_base + (uint32_t)(c32 * 32), r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j++) f[j] = __uint_as_float(r[j]);
          if (live) add_poison(t, k, poison[u & 1], ONE, w, nt, pos, c32 * 32, f);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j++) r[j] = __float_as_uint(f[j]);
          tc_st32(tO + lane_base + (uint32_t)(c32 * 32), r);
        }
        tc_wait_st();
      }
      // Rows leave through 4 KB of shared memory per warp, 128 bytes of each at a time, by one TMA store where the warp's 32 rows are whole tokens of the unit, and
      // otherwise so that a store is four whole lines (a thread per row and store is 32 lines for 512 bytes). Chunk x of row i lies at x ^ (i & 7).
      const bool by_tma = !ONE && np == 1 && 32 % t.G == 0 && __all_sync(0xffffffffu, live);
      uint4* stage = (uint4*)(smem + (NQ + 2 * RING) * TILE) + warp * 256;
      const int64_t to = live ? np > 1 ? (at * np + p) * D * 4 : at * D * 2 : -1;
      auto leave = [&](int piece) {
        uint8_t* dst0 = (np > 1 ? (uint8_t*)t.join.o : (uint8_t*)a.out) + piece * 128 + (lane & 7) * 16;
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const int i = x * 4 + (lane >> 3);
          const int64_t dst = __shfl_sync(0xffffffffu, to, i);
          const uint4 v = stage[i * 8 + ((lane & 7) ^ (i & 7))];
          if (dst >= 0) *(uint4*)(dst0 + dst) = v;
        }
        __syncwarp();
      };
#pragma unroll 1
      for (int h = 0; h < QA; h++) {
        uint32_t r[64];
        if (nt > 0 && any_live) {
          tc_ld32(tO + lane_base + (uint32_t)(h * 64), r);
          tc_ld32(tO + lane_base + (uint32_t)(h * 64 + 32), r + 32);
          tc_wait_ld();
        }
        if (nt > 0 && h == QA - 1) {  // O may be begun anew
          tc_fence_before();
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&o_free[w])) : "memory");
        }
        if (!any_live) continue;
        if (l_run == 0.f) {  // nothing seen
#pragma unroll
          for (int j = 0; j < 64; j++) r[j] = 0;
        }
        if (ONE) {
          if (live && l_run != 0.f) {
            float* dst = t.join.o + (at * np + p) * D + h * 64;
#pragma unroll
            for (int j = 0; j < 64; j += 4) *(uint4*)(dst + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
          }
          __syncwarp();
        } else if (np > 1) {
#pragma unroll
          for (int piece = 0; piece < 2; piece++) {
#pragma unroll
            for (int x = 0; x < 8; x++) {
              const int j = piece * 32 + x * 4;
              stage[lane * 8 + (x ^ (lane & 7))] = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            }
            leave(2 * h + piece);
          }
        } else {
          auto two = [&](int j) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(r[j]) * inv, __uint_as_float(r[j + 1]) * inv);
            return *(const uint32_t*)&v;
          };
#pragma unroll
          for (int x = 0; x < 8; x++) stage[lane * 8 + (x ^ (lane & 7))] = make_uint4(two(x * 8), two(x * 8 + 2), two(x * 8 + 4), two(x * 8 + 6));
          if (by_tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(&map_o), "r"(h * 64), "r"(k.hk * t.G),
                           "r"((int)(k.row0 + tok)), "r"(smem_u32(stage))
                           : "memory");
              asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");  // read before the place is used again
            }
            __syncwarp();
          } else {
            leave(h);
          }
        }
      }
      unit_read(u);
      c += n_all;
    }
    if (!good && lane == 0) set_status(t.status, 45);
  }
  __syncwarp();
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
  // Parts, by key tiles as the unit of time (2.6 us; 1.5 with one tile): rounds of units that are all as long, each with three tiles more for its start and
  // its end, and, where there are several sequences, lengths spread below max_len (mean 0.65): then the longest unit, or what the SMs have to do together.
  // A prompt's rows see half of it. The join costs 4 us and its bytes. (16 sequences of 1.5 to 8 thousand keys, five new tokens, eight heads:
  // one part 121 us, two 84, four 96; one of 16 thousand, 512 new tokens: two 176, three 229, four 193. Calls in a row on the same data; with other data in between two
  // parts take 92 and 200.)
  const double units = (double)std::max<int64_t>((a.at.T + tb - 1) / tb, a.at.B) * a.Hkv, sms = ctx->sm_count;
  const double keys = (double)std::max<int64_t>(1, paged_walk_tiles(a, BKV)), seen = keys * (1 - 0.5 * std::min(1.0, (double)a.max_new / std::max(1, a.max_len)));
  const int outs = ONE ? 2 : 1;
  double best = 1e30;
  t.parts = 1;
  for (int p = 1; p <= 64 && p <= keys; p += p < 8 ? 1 : p / 4) {
    const double out_bytes = (double)a.at.T * a.Hq * p * outs * (64 * QA + 2) * 4;
    if (p > 1 && out_bytes > (double)(256 << 20)) break;
    const double longest = std::ceil(keys / p) + 3, even = std::ceil(units * p / sms) * (std::ceil(seen / p) + 3);
    const double spread = a.at.B > 1 ? std::max(longest, (units * seen * 0.65 + 3 * units * p) / sms) : even;
    const double cost = (even + spread) / 2 + (p * outs > 1 ? (4 + out_bytes / 2.5e6) / (ONE ? 1.5 : 2.6) : 0);
    if (cost < best * 0.98) best = cost, t.parts = p;
  }
  const int np = outs * t.parts;
  if (np > 1) SB_TRY(paged_join_scratch(ctx, a, np, &t.join));
  const int64_t blocks = std::min<int64_t>(tiles * a.Hkv * t.parts, ctx->sm_count);
  t.one_round = tiles * a.Hkv * t.parts <= ctx->sm_count;
  // Sequences of one tile, more of them than the search keeps in registers: in their own order (1000 of at most 60 keys: 640 us searched for, 361 so; 256 of 1 to 2 thousand 474 and 357).
  t.direct = !t.one_round && a.max_new <= tb && a.at.B > 128;
  CUtensorMap mq, mk, mv, mo;
  const int64_t rows = (int64_t)a.at.n_pages * a.Hkv * a.at.page;
  SB_TRY(map_tokens(&mq, a.q, a.at.T, a.Hq, a.D, t.G, t.tw));
  SB_TRY(map_tokens(&mo, a.out, a.at.T, a.Hq, a.D, t.G, std::max(1, 32 / t.G)));  // the rows of a warp
  SB_TRY(paged_map_rows(&mk, a.k, rows, a.D, std::min(a.at.page, BKV)));
  SB_TRY(paged_map_rows(&mv, a.v, rows, a.D, std::min(a.at.page, BKV)));
  constexpr size_t smem = tiles_smem<QA, ONE>();
  static SbDeviceOnce once;  // one per instantiation
  SB_CUDA(once.run(ctx->device, [&] { return cudaFuncSetAttribute(attn_paged_tiles_kernel<QA, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
  SB_CUDA(sb_launch(ctx, attn_paged_tiles_kernel<QA, ONE>, dim3((unsigned)blocks), dim3(THREADS), smem, mq, mk, mv, mo, t));
  ctx->launches++;
  return np > 1 ? paged_join(ctx, a, t.join) : STRICTB200_OK;
}

}  // namespace

int k_attn_paged_tiles(strictb200_ctx* ctx, const PagedAttnArgs& a) {
  // One tile where no sequence has more and the keys are many enough to pay for the join (20 rows: 16 sequences of 8192 keys 134 us with one tile and 161 with two, 256
  // of 1 to 2 thousand 469 and 485, 500 of 200 to 600 702 and 613), and the two shares of all rows take at most 256 MB of scratch.
  const bool one = (int64_t)a.max_new * (a.Hq / a.Hkv) <= BQ && paged_walk_tiles(a, BKV) >= 10 && a.at.T * a.Hq * 2 * (a.D + 2) * 4 <= ((int64_t)256 << 20);
  if (a.D == 128) return one ? launch<2, true>(ctx, a) : launch<2, false>(ctx, a);
  return one ? launch<1, true>(ctx, a) : launch<1, false>(ctx, a);
}
