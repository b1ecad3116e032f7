// Attention over packed prompts on the 5th-generation tensor cores.
//
// Mathematics: per query row, one pass over the keys in tiles of kKeys with the
// running maximum m and sum l of the softmax; O is rescaled when m moves far.
//
// Bound: the tensor cores (4 D flops per visible pair and head) and, next to
// them, the exponentials: those of a tile keep the MUFU as busy as its two
// products keep the tensor core.  So a CTA carries two query tiles, each with
// its own softmax warps and MMA warp, that run past each other freely.
//
// Query tile: 128 rows = R tokens x the G query heads of one kv head (R = 128 /
// G), loaded by one box [R][G][64] per half head, so that k and v are read once
// for the whole group, short prompts fill the tile, and a causal tile spans few
// tokens.  k and v tiles (kKeys tokens) go through a ring of shared-memory slots
// filled by TMA.  TMEM holds, for each query tile, the scores S, the weights P
// (bf16, the A operand of the second product straight from TMEM) and O.  P has
// columns of its own, so that the next scores are computed while the softmax
// works on these; that is what sets kKeys: 80 keys at D = 128 (S 80 + P 40 + O
// 128 columns, twice, of 512), 128 at D = 64.  (1 x 8192 at D = 128, 32 and 8
// heads: 471 us; 128 keys with P over S, whose next products wait for the weights:
// 536 to 569; 64 keys with P over two S in turn, where nothing waits but a product
// takes as long for 64 columns as for 80: 535.)  v is read as it lies (its N side
// contiguous).
//
// One CTA per SM takes items (two query tiles of one kv head) off a common
// counter, the last rows of a sequence first.  Every role runs on into the next
// item as far as its barriers let it: the next q, k and v are on their way while
// the last weights of this item are computed, its scores while its output is
// written.  (A CTA per item spent 13000 cycles of its own before and after its
// tiles: as much as 6 tiles take.)
//
// Few items over long keys are cut instead: the key tiles of all items, in one
// list, go to the CTAs in equal ranges.  An item that lies in one range is
// written as above; of one that lies in several, each CTA leaves its piece (O as
// it is and the rows' m and l, fp32) in the workspace, and prompt_join_kernel
// adds them in the order of the keys, rescaled to the largest m.  (Nothing else may
// use that workspace between the two launches.)
//
// The two tiles' warps that share a scheduler take turns at the exponentials:
// left alone they fall into step, both in the MUFU at half speed and then both
// waiting (1 x 8192: 453 against 526 us).  Computing a part of them on the fma
// pipe instead (2^n times a polynomial) was slower at every part: the two warps
// of a scheduler have no issue slots to spare.
//
// Measured, causal: 1 x 8192 (32 query and 8 kv heads of 128) 453 to 538 us from
// one board to the next (1.0 to 1.2 PFLOP/s), 8 ragged to 700 38 us (fixed cost of
// a call 7, of an item 2 to 4), 4 x 1024 ragged behind 5003 (16, 4, D = 64) 60 to 72
// us from one run to the next.
//
// Warps 0-3 and 4-7: softmax, output (one thread per row of tile 0, 1).  Warp 8:
// TMA; it also clears the rows of the last v tile that lie past the sequence
// (another sequence's values, which a weight of 0 does not stop if they are
// NaN).  Warps 9, 10: MMA of tile 0, 1.  Warp 11: the items.
#pragma once

#include "fp8gq_device.cuh"
#include "tensor_core.cuh"

namespace fp8gq {

// An item whose keys several CTAs share: CTA c of its first piece to `last`.
struct PrSplit {
  int q0, lq, r0, hk;
  int last;                 // -1: none begins in CTA c
  int pad[3];
};

struct PromptParams {
  __nv_bfloat16* out;
  float* lse;
  int64_t o_token, o_head;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, Tq, Tk, Hq, Hkv;
  int group, rows;          // query heads per kv head; tokens per query tile
  int group_inv;            // 65536 / group, rounded up: x / group = x * group_inv >> 16 for x < 128
  int* counters;            // [2], zero between launches: the next item, the CTAs that are done
  float scale_log2;         // |scale| log2(e)
  int negate;               // scale < 0
  int causal;
  int split;                // equal ranges of key tiles instead of whole items
  PrSplit* splits;          // [grid]
  float* parts;             // [grid][2][PrCfg::kPart]: the piece that a CTA's range begins, ends with
};

constexpr int kPrThreads = 384;

template <int D>
struct PrCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kKeys = D == 128 ? 80 : 128;        // keys per tile
  static constexpr int kQTile = kHalves * 128 * 128;       // bytes of a q tile
  static constexpr int kHalf = kKeys * 128;                // bytes of half a k or v tile (64 values)
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kSlots = D == 128 ? 6 : 8;          // ring slots: k and v tiles in turn
  static constexpr int kStage = 2 * 128 * 128;             // output on its way out: 64 values of each row
  static constexpr size_t kSmem = 1024 + 2 * static_cast<size_t>(kQTile) + kStage + kSlots * static_cast<size_t>(kTile);
  // TMEM columns: O0 O1 S0 S1 P0 P1
  static constexpr int kS = 2 * D, kP = kS + 2 * kKeys, kPCols = (kKeys / 2 + 15) / 16 * 16;
  static_assert(kP + 2 * kPCols <= 512, "TMEM");
  // a piece's result: [2 query tiles][D / 4][128 rows][4] O, then [2][128] (m, l)
  static constexpr int kPartO = 2 * 128 * D, kPart = kPartO + 2 * 128 * 2;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// 128-byte-swizzled operand: K side contiguous (q, k: 8-row groups 1024 bytes
// apart) or N side contiguous (v: groups of 8 tokens 1024 bytes apart, groups
// of 64 values lbo bytes apart).
__device__ __forceinline__ uint64_t pr_desc(uint32_t addr, uint32_t lbo) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// kind::f16, bf16 operands, fp32 sums; M = 128.
__device__ __forceinline__ uint32_t pr_idesc(int n, bool b_n_major, bool negate_a) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (negate_a ? 1u << 13 : 0u) | (b_n_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}

#define FP8GQ_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define FP8GQ_I8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])

// Columns of this warp's 32 lanes.  Loaded registers are valid after
// tmem_wait_ld; tmem_loaded keeps their use behind it.
__device__ __forceinline__ void tmem_ld16r(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : FP8GQ_R8(r, 0), FP8GQ_R8(r, 8)
      : "r"(addr)
      : "memory");
}
#define FP8GQ_B8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
__device__ __forceinline__ void tmem_loaded16(uint32_t* r) { asm volatile("" : FP8GQ_B8(r, 0), FP8GQ_B8(r, 8)::"memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::FP8GQ_I8(r, 0),
      FP8GQ_I8(r, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::FP8GQ_I8(r, 0), "r"(addr)
               : "memory");
}
#undef FP8GQ_B8
#undef FP8GQ_R8
#undef FP8GQ_I8
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kPassAfter = 2;      // 16-key chunks after which the turn is passed

// One lane of the (converged) warp.  tcgen05.mma takes its operands from uniform
// registers; behind a branch on the lane number the compiler issues it lane by
// lane, 114 cycles each, whatever its size (70 to 87 behind this one at 128 x 128
// x 16).
__device__ __forceinline__ bool pr_elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(one));
  return one != 0;
}

// A bounded wait, by one thread, or by all lanes of a warp with one outcome.
__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity) { return mbar_wait_short(bar, parity, kSitePrompt); }
__device__ __forceinline__ bool pr_wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, pr_wait(bar, parity)) != 0;
}

// An item: two query tiles of one sequence and kv head.
struct PrWork {
  int q0, lq, k0, lk;       // the sequence's tokens (q0 < 0: no more items)
  int r0;                   // first token of the item within the sequence
  int hk;
  int n[2];                 // key tiles that the last row of each query tile sees
  int part;                 // >= 0: a piece, whose result goes there
};
constexpr int kPrItems = 2;      // items looked up ahead
// What an item's start and end count in its range, in key tiles (4 x 1024 ragged
// behind 5003, D = 64, and 1 x 4096, 2 kv heads: 2: 59 and 51 us, 4: 61 and 49,
// 8: 64 and 52), and the least range (4 x 16 behind 4000: 6: 25 us, 10: 28, 16:
// 35; above kPrItemCost, so that no range is an item's start alone).
constexpr int kPrItemCost = 4;
constexpr int kPrMinTiles = 6;
static_assert(kPrMinTiles > kPrItemCost, "");

template <int D>
__global__ void __launch_bounds__(kPrThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap tq,
                                                                          const __grid_constant__ CUtensorMap tk,
                                                                          const __grid_constant__ CUtensorMap tv,
                                                                          const PromptParams p) {
  using Cfg = PrCfg<D>;
  constexpr int kSlots = Cfg::kSlots, kTile = Cfg::kTile, kKeys = Cfg::kKeys;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t b_item[kPrItems], b_taken[kPrItems];   // an item is there; every role has it behind it
  __shared__ uint64_t b_want;                                // an item's loads are all on their way: time for the next
  __shared__ uint64_t b_q, b_qfree, b_tail;                  // q is there; q is read; the last v tile is there
  __shared__ uint64_t b_full[kSlots], b_free[kSlots];
  __shared__ uint64_t b_s[2], b_r[2], b_p[2], b_o[2];        // scores ready, read; weights ready; O updated
  __shared__ uint64_t b_out[2];                              // O read
  __shared__ uint64_t b_end[2];                              // at the end: the products issued are done
  __shared__ uint64_t b_turn[2][4];                          // tile i's warp may have the MUFU
  __shared__ uint32_t s_tmem;
  __shared__ PrWork s_work[kPrItems];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t out_stage = base + 2 * Cfg::kQTile;
  const uint32_t ring = out_stage + Cfg::kStage;

  if (warp == 8) {
    if (lane == 0) {
      prefetch_tensormap(&tq);
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
      for (int i = 0; i < kPrItems; ++i) {
        mbar_init(&b_item[i], 1);
        mbar_init(&b_taken[i], 11);       // TMA, 2 MMA, 8 softmax warps
      }
      mbar_init(&b_want, 1);
      mbar_init(&b_q, 1);
      mbar_init(&b_qfree, 2);             // both MMA warps
      mbar_init(&b_tail, 1);
      for (int i = 0; i < kSlots; ++i) {
        mbar_init(&b_full[i], 1);
        mbar_init(&b_free[i], 2);         // both MMA warps
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&b_s[i], 1);
        mbar_init(&b_r[i], 4);            // softmax warps
        mbar_init(&b_p[i], 4);
        mbar_init(&b_o[i], 1);
        mbar_init(&b_out[i], 4);
        mbar_init(&b_end[i], 1);
        for (int x = 0; x < 4; ++x) mbar_init(&b_turn[i][x], 1);
      }
      fence_mbar_init();
    }
  } else if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  grid_dependency_wait();
  bool ok = true;

  // The items as every role sees them; k and v tiles and steps are numbered
  // through all items.
  int item = 0;
  PrWork w;
  auto next_item = [&]() {
    ok = pr_wait_warp(&b_item[item % kPrItems], (item / kPrItems) & 1) && ok;
    if (!ok) return false;
    w = s_work[item % kPrItems];
    return w.q0 >= 0;
  };
  auto leave_item = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&b_taken[item % kPrItems]);
    ++item;
  };

  if (warp >= 8) {
    if (warp == 11) {
      // ---- items ----
      const int span = 2 * p.rows;
      const int share = (p.B + 31) / 32;
      const int b_lo = min(lane * share, p.B), b_hi = min(b_lo + share, p.B);
      auto tokens = [&](int b, int& q0, int& q1, bool record) {
        q0 = __ldg(p.cu_q + b);
        q1 = __ldg(p.cu_q + b + 1);
        if (q0 < 0 || q0 > p.Tq || q1 < q0 || q1 > p.Tq) {
          if (record) record_error(kSiteBadIndex);
          q0 = min(max(q0, 0), p.Tq);
          q1 = min(max(q1, q0), p.Tq);
        }
      };
      auto keys = [&](int b, int& k0, int& k1) {
        k0 = __ldg(p.cu_k + b);
        k1 = __ldg(p.cu_k + b + 1);
        if (k0 < 0 || k0 > p.Tk || k1 < k0 || k1 > p.Tk) {
          record_error(kSiteBadIndex);
          k0 = min(max(k0, 0), p.Tk);
          k1 = min(max(k1, k0), p.Tk);
        }
      };
      // key tiles that the query tiles of the item at token r0 see
      auto seen_tiles = [&](int r0, int lq, int lk, int* n) {
        for (int i = 0; i < 2; ++i) {
          const int end = min(r0 + (i + 1) * p.rows, lq);          // past the query tile's last token
          int seen = end > r0 + i * p.rows ? lk : 0;
          if (p.causal && seen) seen = min(lk, max(0, end + lk - lq));
          n[i] = (seen + kKeys - 1) / kKeys;
        }
      };
      int it = 0;
      auto post = [&](const PrWork& x, bool writer) {              // the next item, or the end
        if (it >= kPrItems) ok = pr_wait_warp(&b_taken[it % kPrItems], (it / kPrItems - 1) & 1);
        if (!ok) return;
        if (writer) s_work[it % kPrItems] = x;
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_item[it % kPrItems]);
        ++it;
      };
      int mine = 0;
      for (int b = b_lo; b < b_hi; ++b) {
        int q0, q1;
        tokens(b, q0, q1, blockIdx.x == 0);
        mine += (q1 - q0 + span - 1) / span;
      }
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const int tiles = __shfl_sync(0xffffffffu, incl, 31), total = tiles * p.Hkv;
      PrWork x;
      x.q0 = -1;
      x.part = -1;
      if (p.split) {
        // ---- equal ranges: lane b has sequence b ----
        int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
        if (lane < p.B) {
          tokens(lane, q0, q1, false);
          keys(lane, k0, k1);
        }
        const int lq = q1 - q0, lk = k1 - k0;
        // this lane's tile of the 32 from `from` on; what an item of it counts
        int yb, ynb, yn[2];
        auto look = [&](int from) {
          const int t = from + lane;
          yb = 0;
#pragma unroll
          for (int o = 16; o; o >>= 1) yb += __shfl_sync(0xffffffffu, incl, yb + o - 1) <= t ? o : 0;
          const int at = __shfl_sync(0xffffffffu, incl - mine, yb), nb = __shfl_sync(0xffffffffu, mine, yb);
          const int ylq = __shfl_sync(0xffffffffu, lq, yb), ylk = __shfl_sync(0xffffffffu, lk, yb);
          ynb = (nb - 1 - (t - at)) * span;                        // its first token
          if (t >= tiles) return 0;
          seen_tiles(ynb, ylq, ylk, yn);
          return max(yn[0], yn[1]) + kPrItemCost;
        };
        int64_t work = 0;
        for (int from = 0; from < tiles; from += 32) work += __reduce_add_sync(0xffffffffu, static_cast<unsigned>(look(from)));
        work *= p.Hkv;
        const int64_t ctas = max(min(static_cast<int64_t>(gridDim.x), work / kPrMinTiles), static_cast<int64_t>(1));
        const int cta = static_cast<int>(blockIdx.x);
        const int64_t lo = cta < ctas ? work * cta / ctas : work, hi = cta < ctas ? work * (cta + 1) / ctas : work;
        PrSplit mark{};
        mark.last = -1;
        int64_t at = 0;
        for (int from = 0; from < tiles && at < hi && ok; from += 32) {
          const int cost = look(from);
          int sum = cost;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
          }
          const int64_t a0 = at + static_cast<int64_t>(sum - cost) * p.Hkv, a1 = at + static_cast<int64_t>(sum) * p.Hkv;
          at = __shfl_sync(0xffffffffu, a1, 31);
          uint32_t in = __ballot_sync(0xffffffffu, cost > 0 && a0 < hi && a1 > lo);
          for (; in && ok; in &= in - 1) {
            const int from_lane = __ffs(in) - 1;
            const int64_t a = __shfl_sync(0xffffffffu, a0, from_lane);
            const int c = __shfl_sync(0xffffffffu, cost, from_lane), n = c - kPrItemCost;
            const int b = __shfl_sync(0xffffffffu, yb, from_lane), r0 = __shfl_sync(0xffffffffu, ynb, from_lane);
            const int n0 = __shfl_sync(0xffffffffu, yn[0], from_lane), n1 = __shfl_sync(0xffffffffu, yn[1], from_lane);
            const int xq0 = __shfl_sync(0xffffffffu, q0, b), xlq = __shfl_sync(0xffffffffu, lq, b);
            const int xk0 = __shfl_sync(0xffffffffu, k0, b), xlk = __shfl_sync(0xffffffffu, lk, b);
            for (int hk = lo > a ? static_cast<int>((lo - a) / c) : 0; hk < p.Hkv && a + static_cast<int64_t>(hk) * c < hi && ok; ++hk) {
              const int64_t first = a + static_cast<int64_t>(hk) * c + kPrItemCost;      // its first key tile
              const int j0 = static_cast<int>(min(max(lo - first, static_cast<int64_t>(0)), static_cast<int64_t>(n)));
              const int j1 = static_cast<int>(min(max(hi - first, static_cast<int64_t>(0)), static_cast<int64_t>(n)));
              // an item without keys belongs to the range that it begins in
              if (j0 == j1 && (n > 0 || first - kPrItemCost < lo)) continue;
              x.q0 = xq0;
              x.lq = xlq;
              x.k0 = xk0 + j0 * kKeys;
              x.lk = xlk - j0 * kKeys;
              x.r0 = r0;
              x.hk = hk;
              x.n[0] = max(min(n0, j1) - j0, 0);
              x.n[1] = max(min(n1, j1) - j0, 0);
              x.part = j1 - j0 == n ? -1 : 2 * cta + (j0 == 0 ? 1 : 0);
              if (x.part >= 0 && j0 == 0) {
                mark = PrSplit{xq0, xlq, r0, hk, static_cast<int>(((first + n) * ctas - 1) / work), {}};
              }
              post(x, lane == 0);
            }
          }
        }
        if (lane == 0) p.splits[cta] = mark;
        x.q0 = -1;
        if (ok) post(x, lane == 0);
      } else {
        int id = blockIdx.x;                          // the first item; the others off the counter
        for (;;) {
          x.q0 = -1;
          const int tile = id / p.Hkv;
          const bool here = id < total && tile < incl && tile >= incl - mine;
          if (here) {
            int at = incl - mine;
            for (int b = b_lo; b < b_hi; ++b) {
              int q0, q1;
              tokens(b, q0, q1, false);
              const int nb = (q1 - q0 + span - 1) / span;
              if (tile < at + nb) {
                int k0, k1;
                keys(b, k0, k1);
                x.q0 = q0;
                x.lq = q1 - q0;
                x.k0 = k0;
                x.lk = k1 - k0;
                x.hk = id - tile * p.Hkv;
                x.r0 = (nb - 1 - (tile - at)) * span;
                seen_tiles(x.r0, x.lq, x.lk, x.n);
                break;
              }
              at += nb;
            }
          }
          post(x, here || (lane == 0 && id >= total));
          if (!ok || id >= total) break;
          // not before this item's loads are issued: an item taken early is one that
          // an idle CTA cannot take
          ok = pr_wait_warp(&b_want, (it - 1) & 1);
          if (!ok) break;
          if (lane == 0) id = gridDim.x + atomicAdd(p.counters, 1);
          id = __shfl_sync(0xffffffffu, id, 0);
        }
      }
      // the last CTA to get here leaves the counters as it found them
      if (lane == 0 && !p.split) {
        __threadfence();
        if (atomicAdd(p.counters + 1, 1) == static_cast<int>(gridDim.x) - 1) {
          p.counters[0] = 0;
          p.counters[1] = 0;
        }
      }
    } else if (warp == 8) {
      // ---- TMA ----
      int x0 = 0, items = 0, tails = 0;             // k and v tiles, items and tails so far
      int q_sent = 0, sent = 0;                     // q, k and v tiles on their way or there
      bool tail_sent = false;                       // the last of them is a v tile whose copy b_tail counts
      while (next_item()) {
        const int n = max(w.n[0], w.n[1]);
        const bool partial = n * kKeys > w.lk;      // the last tile reaches past the sequence
        if (n > 0) {
          if (items > 0) ok = pr_wait_warp(&b_qfree, (items - 1) & 1);
          if (!ok) break;
          ++q_sent;
          if (pr_elect()) {
            mbar_arrive_expect_tx(&b_q, 2 * Cfg::kHalves * p.group * p.rows * 128);
            for (int i = 0; i < 2; ++i)
              for (int h = 0; h < Cfg::kHalves; ++h)
                tma_load_3d(base + i * Cfg::kQTile + h * 16384, &tq, 64 * h, w.hk * p.group, w.q0 + w.r0 + i * p.rows, &b_q);
          }
          __syncwarp();
          for (int i = 0; i < 2 * n; ++i) {                    // k and v tiles in turn
            const int x = x0 + i, slot = x % kSlots;
            if (x >= kSlots) ok = pr_wait_warp(&b_free[slot], (x / kSlots - 1) & 1);
            if (!ok) break;
            ++sent;
            tail_sent = partial && i == 2 * n - 1;
            if (pr_elect()) {
              uint64_t* bar = tail_sent ? &b_tail : &b_full[slot];
              mbar_arrive_expect_tx(bar, kTile);
              for (int h = 0; h < Cfg::kHalves; ++h)
                tma_load_3d(ring + slot * kTile + h * Cfg::kHalf, (i & 1) ? &tv : &tk, 64 * h, w.hk, w.k0 + (i >> 1) * kKeys, bar);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (partial) {
            // rows past the sequence: zeros, then the tile is there
            const int slot = (x0 + 2 * n - 1) % kSlots, valid = w.lk - (n - 1) * kKeys;
            ok = pr_wait_warp(&b_tail, tails & 1);
            if (!ok) break;
            for (int x = valid * 8 + lane; x < kKeys * 8; x += 32)
              for (int h = 0; h < Cfg::kHalves; ++h)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + slot * kTile + h * Cfg::kHalf + x * 16), "r"(0u)
                             : "memory");
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_full[slot]);
            tail_sent = false;
            ++tails;
          }
          x0 += 2 * n;
          ++items;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_want);
        leave_item();
      }
      // every copy has landed before the CTA ends, whichever role gave a wait up
      // (where none did, every tile is used and this waits for nothing else)
      if (lane == 0) {
        if (q_sent) pr_wait(&b_q, (q_sent - 1) & 1);
        for (int x = max(sent - kSlots, 0); x < sent; ++x) {
          if (tail_sent && x == sent - 1) pr_wait(&b_tail, tails & 1);
          else pr_wait(&b_full[x % kSlots], (x / kSlots) & 1);
        }
      }
    } else {
      // ---- MMA of tile i: the warp waits together, one lane issues ----
      const int i = __shfl_sync(0xffffffffu, warp, 0) - 9;
      const uint32_t id_s = pr_idesc(kKeys, false, p.negate != 0), id_o = pr_idesc(D, true, false);
      const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t ts = t0 + Cfg::kS + i * kKeys, tp = t0 + Cfg::kP + i * Cfg::kPCols, to = t0 + i * D;
      int x0 = 0, items = 0, step0 = 0, outs = 0;   // tiles, items with tiles, this tile's steps and outputs so far
      auto full = [&](int x) { return pr_wait_warp(&b_full[x % kSlots], (x / kSlots) & 1); };
      auto scores = [&](int j) {                           // S = Q K^T of tile j
        const int x = x0 + 2 * j, step = step0 + j;
        ok = full(x) && (step == 0 || pr_wait_warp(&b_r[i], (step - 1) & 1));
        if (!ok) return;
        tc_fence_after();
        const uint32_t a = base + i * Cfg::kQTile, b = ring + (x % kSlots) * kTile;
        if (pr_elect()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(ts, pr_desc(a + (k >> 2) * 16384 + (k & 3) * 32, 16), pr_desc(b + (k >> 2) * Cfg::kHalf + (k & 3) * 32, 16),
                   id_s, k > 0);
          mma_commit(&b_s[i]);
          mma_commit(&b_free[x % kSlots]);
        }
        __syncwarp();
      };
      while (next_item()) {
        const int mine = w.n[i], n = max(w.n[0], w.n[1]);
        if (n > 0) {
          ok = pr_wait_warp(&b_q, items & 1);
          if (ok && mine > 0) scores(0);
          for (int j = 0; j < mine && ok; ++j) {
            const bool more = j + 1 < mine;
            if (more) {
              scores(j + 1);
              if (!ok) break;
            }
            const int x = x0 + 2 * j + 1;
            ok = full(x) && (j > 0 || outs == 0 || pr_wait_warp(&b_out[i], (outs - 1) & 1)) &&
                 pr_wait_warp(&b_p[i], (step0 + j) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b = ring + (x % kSlots) * kTile;              // O += P V
            if (pr_elect()) {
              if (!more) mma_commit(&b_qfree);                           // q has been read
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k) mma_ts(to, tp + 8 * k, pr_desc(b + k * 2048, Cfg::kHalf), id_o, j > 0 || k > 0);
              mma_commit(&b_free[x % kSlots]);
              mma_commit(&b_o[i]);                                       // (the last commit of an item)
            }
            __syncwarp();
          }
          if (mine == 0 && ok && lane == 0) mbar_arrive(&b_qfree);
          // the tiles that only the other query tile sees
          for (int x = 2 * mine; x < 2 * n && ok; ++x) {
            ok = full(x0 + x);
            if (ok && lane == 0) mbar_arrive(&b_free[(x0 + x) % kSlots]);
          }
          ++items;
        }
        if (!ok) break;
        x0 += 2 * n;
        step0 += mine;
        if (mine > 0) ++outs;
        leave_item();
      }
      // what has been issued completes before the CTA ends, whichever role gave up
      if (pr_elect()) mma_commit(&b_end[i]);
      __syncwarp();
      pr_wait_warp(&b_end[i], 0);
    }
  } else {
    // ---- softmax and output: one thread per row ----
    const int i = warp >> 2, row = tid & 127;
    const int row_tok = (row * p.group_inv) >> 16, row_head = row - row_tok * p.group;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t ts = lanes + Cfg::kS + i * kKeys, tp = lanes + Cfg::kP + i * Cfg::kPCols, to = lanes + i * D;
    const uint32_t stage = out_stage + warp * 4096;        // 32 rows of 64 values
    const float c = p.scale_log2;
    int step0 = 0, turns = 0;                              // this tile's steps so far, the turns of both
    auto take_turn = [&]() { return (i == 0 && turns == 0) || pr_wait_warp(&b_turn[i][warp & 3], (turns - 1 + i) & 1); };
    auto pass_turn = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&b_turn[1 - i][warp & 3]);
      ++turns;
    };
    while (next_item()) {
      const int mine = w.n[i];
      const int tok = w.r0 + i * p.rows + row_tok;         // token within the sequence
      const bool live = row_tok < p.rows && tok < w.lq;
      int lim = w.lk;                                      // keys this row sees
      if (p.causal) lim = max(0, min(w.lk, tok + 1 + w.lk - w.lq));
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < mine; ++j) {
        const int step = step0 + j;
        ok = pr_wait_warp(&b_s[i], step & 1);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[kKeys];
#pragma unroll
        for (int x = 0; x < kKeys; x += 16) tmem_ld16r(ts + x, s + x);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < kKeys; x += 16) tmem_loaded16(s + x);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_r[i]);               // the next scores may come
        const int vis = lim - j * kKeys;
        if (__any_sync(0xffffffffu, vis < kKeys)) {
#pragma unroll
          for (int x = 0; x < kKeys; ++x)
            if (x >= vis) s[x] = 0xff800000u;
        }
        float mx8[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) mx8[y] = fmaxf(__uint_as_float(s[y]), __uint_as_float(s[8 + y]));
#pragma unroll
        for (int x = 16; x < kKeys; x += 16)
#pragma unroll
          for (int y = 0; y < 8; ++y) mx8[y] = fmaxf(fmaxf(mx8[y], __uint_as_float(s[x + y])), __uint_as_float(s[x + 8 + y]));
        const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])), fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
        // O keeps its reference maximum until a row's weights would pass 2^8: they are
        // as exact at any scale, but O has to stay in fp32's range with them
        const bool move = (mx - m) * c > 8.0f || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float mn = fmaxf(m, mx);
          if (j > 0) {
            // (the products of the tile before have updated O)
            ok = pr_wait_warp(&b_o[i], (step - 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const float a = m == -INFINITY ? 0.0f : ex2f((m - mn) * c);
            l *= a;
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
              uint32_t o[16];
              tmem_ld16r(to + x, o);
              tmem_wait_ld();
              tmem_loaded16(o);
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * a);
              tmem_st16(to + x, o);
            }
          }
          m = mn;
        }
        const float mc = m == -INFINITY ? 0.0f : m * c;
        // weights in bf16, v's type, as the two operands of a product have one type:
        // half an ulp each (more bits would take a second product); l sums the unrounded
        const float2 c2 = make_float2(c, c), mc2 = make_float2(-mc, -mc);
        float2 sum[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) sum[y] = make_float2(0.0f, 0.0f);
        if (step > 0) {
          // the products of the tile before have read P by now
          ok = pr_wait_warp(&b_o[i], (step - 1) & 1);
          if (!ok) break;
          tc_fence_after();
        }
        ok = take_turn();
        if (!ok) break;
#pragma unroll
        for (int x = 0; x < kKeys; x += 16) {
          uint32_t q[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const float2 t = fma2(make_float2(__uint_as_float(s[x + 2 * y]), __uint_as_float(s[x + 2 * y + 1])), c2, mc2);
            const float2 e = make_float2(ex2f(t.x), ex2f(t.y));
            sum[y & 3] = add2(sum[y & 3], e);
            const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
            q[y] = *reinterpret_cast<const uint32_t*>(&h);
          }
          tmem_st8(tp + x / 2, q);
          if (x / 16 == kPassAfter) pass_turn();           // (the hand-over takes as long as the rest)
        }
        const float2 sum2 = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
        l += sum2.x + sum2.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_p[i]);
      }
      for (int j = mine; j < max(w.n[0], w.n[1]) && ok; ++j) {       // the other tile's last turns
        ok = take_turn();
        pass_turn();
      }
      if (!ok) break;
      step0 += mine;
      if (mine > 0) {
        ok = pr_wait_warp(&b_o[i], (step0 - 1) & 1);
        if (!ok) break;
        tc_fence_after();
      }
      if (w.part >= 0) {
        // a piece: O as it is, and its (m, l), of the rows that there are
        float* part = p.parts + static_cast<int64_t>(w.part) * Cfg::kPart;
        if (mine > 0) {
#pragma unroll 1
          for (int x = 0; x < D; x += 16) {
            uint32_t o[16];
            tmem_ld16r(to + x, o);
            tmem_wait_ld();
            tmem_loaded16(o);
            if (!live) continue;
#pragma unroll
            for (int y = 0; y < 16; y += 4)
              *reinterpret_cast<uint4*>(part + ((i * (D / 4) + (x + y) / 4) * 128 + row) * 4) =
                  make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b_out[i]);
        }
        if (live) *reinterpret_cast<float2*>(part + Cfg::kPartO + (i * 128 + row) * 2) = make_float2(m, l);
        leave_item();
        continue;
      }
      const float r = l > 0.0f ? 1.0f / l : l;             // a row that sees nothing: 0; NaN stays
      // 64 values of each row at a time through shared memory (chunks swizzled
      // by row), so that the warp writes whole rows
#pragma unroll 1
      for (int half = 0; half < Cfg::kHalves; ++half) {
        __syncwarp();                                      // the half before is on its way
#pragma unroll
        for (int q = 0; q < 64; q += 16) {
          uint32_t o[16];
          if (mine > 0) {
            tmem_ld16r(to + 64 * half + q, o);
            tmem_wait_ld();
            tmem_loaded16(o);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t hw[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float v0 = l == 0.0f ? 0.0f : __uint_as_float(o[8 * x + 2 * z]) * r;
              const float v1 = l == 0.0f ? 0.0f : __uint_as_float(o[8 * x + 2 * z + 1]) * r;
              const __nv_bfloat162 b = __floats2bfloat162_rn(v0, v1);
              hw[z] = *reinterpret_cast<const uint32_t*>(&b);
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((q / 8 + x) ^ (lane & 7)) * 16),
                         "r"(hw[0]), "r"(hw[1]), "r"(hw[2]), "r"(hw[3]) : "memory");
          }
        }
        if (half == Cfg::kHalves - 1 && mine > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b_out[i]);           // O may be overwritten
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int rr = 4 * x + (lane >> 3), ch = lane & 7;           // row within the warp, chunk
          const int rt = (((warp & 3) * 32 + rr) * p.group_inv) >> 16, rh = (warp & 3) * 32 + rr - rt * p.group;
          const int tt = w.r0 + i * p.rows + rt;
          if (rt < p.rows && tt < w.lq) {
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(stage + rr * 128 + (ch ^ (rr & 7)) * 16) : "memory");
            *reinterpret_cast<uint4*>(p.out + (static_cast<int64_t>(w.q0) + tt) * p.o_token +
                                      (w.hk * p.group + rh) * p.o_head + 64 * half + 8 * ch) = v;
          }
        }
      }
      if (live && p.lse)
        p.lse[(static_cast<int64_t>(w.q0) + tok) * p.Hq + w.hk * p.group + row_head] =
            l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m * c) + log2f(l)) * 0.6931471805599453f;
      leave_item();
    }
    tmem_wait_st();                                        // (stores of a step that was given up)
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  grid_launch_dependents();
}

// Joins the pieces of the items that several CTAs share, in the order of the
// keys.  Block (c, x): the item that begins in CTA c and goes on, values 16 x to
// 16 x + 15; warp: 32 rows, one per lane.
template <int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptParams p) {
  using Cfg = PrCfg<D>;
  grid_dependency_wait();
  const int c = blockIdx.x, d0 = 16 * blockIdx.y;
  const PrSplit e = p.splits[c];
  // (records that something else has written to the workspace between the two
  // launches, against the rule, do not become addresses)
  const bool good = e.last < static_cast<int>(gridDim.x) && e.q0 >= 0 && e.lq >= 0 && e.lq <= p.Tq - e.q0 && e.r0 >= 0 &&
                    e.r0 <= e.lq && e.hk >= 0 && e.hk < p.Hkv;
  if (e.last > c && !good) record_error(kSiteBadIndex);
  if (e.last > c && good) {
    const int i = threadIdx.x >> 7, row = threadIdx.x & 127;
    const int row_tok = (row * p.group_inv) >> 16, row_head = row - row_tok * p.group;
    const int tok = e.r0 + i * p.rows + row_tok;
    if (row_tok < p.rows && tok < e.lq) {
      const float* ml = p.parts + Cfg::kPartO + (i * 128 + row) * 2;
      const float* po = p.parts + ((i * (D / 4) + d0 / 4) * 128 + row) * 4;
      auto slot = [&](int k) { return static_cast<int64_t>(2 * k + (k == c ? 1 : 0)) * Cfg::kPart; };
      float m = -INFINITY;
#pragma unroll 4
      for (int k = c; k <= e.last; ++k) m = fmaxf(m, ml[slot(k)]);
      float l = 0.0f, acc[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) acc[y] = 0.0f;
#pragma unroll 2
      for (int k = c; k <= e.last; ++k) {
        const float2 r = *reinterpret_cast<const float2*>(ml + slot(k));
        float4 o[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) o[y] = *reinterpret_cast<const float4*>(po + slot(k) + y * 512);
        // a row that saw nothing there left no O; NaN stays
        const bool none = r.x == -INFINITY && r.y == 0.0f;
        const float a = r.x == -INFINITY ? 1.0f : ex2f((r.x - m) * p.scale_log2);
        if (!none) {
          l = fmaf(r.y, a, l);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            acc[4 * y] = fmaf(o[y].x, a, acc[4 * y]);
            acc[4 * y + 1] = fmaf(o[y].y, a, acc[4 * y + 1]);
            acc[4 * y + 2] = fmaf(o[y].z, a, acc[4 * y + 2]);
            acc[4 * y + 3] = fmaf(o[y].w, a, acc[4 * y + 3]);
          }
        }
      }
      const float r = l > 0.0f ? 1.0f / l : l;
      uint32_t h[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(l == 0.0f ? 0.0f : acc[2 * y] * r, l == 0.0f ? 0.0f : acc[2 * y + 1] * r);
        h[y] = *reinterpret_cast<const uint32_t*>(&b);
      }
      const int64_t t = static_cast<int64_t>(e.q0) + tok;
      const int head = e.hk * p.group + row_head;
      uint4* out = reinterpret_cast<uint4*>(p.out + t * p.o_token + head * p.o_head + d0);
      out[0] = make_uint4(h[0], h[1], h[2], h[3]);
      out[1] = make_uint4(h[4], h[5], h[6], h[7]);
      if (d0 == 0 && p.lse)
        p.lse[t * p.Hq + head] =
            l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m * p.scale_log2) + log2f(l)) * 0.6931471805599453f;
    }
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
