// Attention of one new token per sequence over a paged key-value cache.
//
// Mathematics: o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q.k_j,
// in one pass over the cache with the running maximum m; partial results
// (m, l, o) of disjoint token ranges join by rescaling to the larger maximum.
//
// Bound: HBM, every cached byte read once (16 flops per byte at most, with the
// heads padded to the matrix instruction's 8 columns).
//
// Work split: the tiles (4 warps x kTok tokens of one sequence and kv head) of
// all sequences form one flat list, cut into equal contiguous ranges, one per
// CTA, two CTAs per SM; the start of each (sequence, head) counts as
// kDecItemCost tiles more.  The lengths are read on the device (a captured step
// replays while they grow), so ragged batches and long single sequences
// balance the same way.  A (sequence, head) that lies in several ranges leaves
// partial results in the workspace; the last CTA to arrive joins them in range
// order, so the result does not depend on who is last.
//
// Inside a CTA each warp runs alone: its lanes look up the pages of its own
// kTok tokens and copy their rows of k and v (8 KB per step; while one of the
// kDecStages is computed the other two are on their way), and it computes on
// them with matrix instructions whose M side is the tokens (S^T = K Q^T, 16 x 8)
// and then the head's values (O^T = V^T P^T), so a group of up to 8 query heads
// wastes nothing of K and V and no barrier stands in the loop.  The copies are
// 16-byte cp.async: any page size and stride, and one bulk copy per row was
// measured at 16 cycles each (8 x 32768 tokens, e4m3: 235 us against 131 as the
// rest stood then).
//
// Measured in a CUDA graph, 32 query and 8 kv heads of 128: 64 x 4096 tokens 184 us
// (5.8 TB/s), 48 ragged to 6000 71 us (5.5 TB/s), 8 x 32768 in e4m3 97 us (5.5
// TB/s), 1 x 333 8.3 us (the latency of one range and its join).  More than 8 heads
// a group, 10 x 1333 (16, 1, 128): 13.1 us in bf16 and in e4m3 (that build spills 208
// bytes); 64 x 4096 (32, 2, 128): 59 us in bf16, 47 in e4m3, where conversions bound it.
#pragma once

#include "fp8gq_device.cuh"
#include "rope_append.cuh"
#include "tensor_core.cuh"

namespace fp8gq {

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_token, q_head;
  CacheView cache;
  const int32_t* table;
  int64_t ld_table;
  int max_pages;
  int page_shift;           // log2(page_size), or -1
  const int32_t* lens;
  __nv_bfloat16* out;
  int64_t o_token, o_head;
  float* lse;
  int B, Hq, Hkv;
  int group;                // query heads per kv head
  int blocks;               // head blocks (of 8 kNT query heads) per kv head
  float scale_log2;         // softmax scale * log2(e) (* k_scale)
  float out_scale;          // v_scale
  int* counters;            // [grid], zero between launches
  float* partials;          // [grid][2][kSlot]
};

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecStages = 3;
constexpr int kDecCtas = 2;                 // per SM (of 4 KB steps, four: 128 x 2047 e4m3, D = 64, 36 us against 25)
constexpr int kDecCounterBytes = 16384;     // the workspace's counters (the tile kernel's too)
// Tiles per CTA below which fewer CTAs work (1 x 333 and 1 x 2000 tokens: 1: 8.2
// and 11.3 us; 2: 8.6 and 9.5; 3: 9.7 and 10.6).
constexpr int kDecMinTiles = 2;
// What starting a (sequence, head) counts, in tiles (48 ragged to 6000: 0: 108
// us, 1: 75, 2: 71).
constexpr int kDecItemCost = 2;

template <int D, bool kFp8, int kNT>
struct DecCfg {
  static constexpr int kStep = 8192;                    // bytes of k and v rows of one warp's step
  static constexpr int kRow = D * (kFp8 ? 1 : 2);       // bytes of a row
  static constexpr int kTok = kStep / 2 / kRow;
  static constexpr int kTile = kTok * kDecWarps;
  static constexpr int kChunks = kRow / 16;
  // distance of rows in shared memory: rows read by one phase of a load fall on
  // different banks (the e4m3 k rows: pairs of rows meet, two phases more)
  static constexpr int kRowK = kFp8 ? kRow : kRow + 16;
  static constexpr int kRowV = kRow + 16;
  static constexpr int kStage = kTok * (kRowK + kRowV);
  static constexpr int kPad = D + 4;                    // o in shared memory: conflict-free fragment writes
  static_assert(kStage >= 8 * kNT * kPad * 4 && kStage % 16 == 0, "a warp's o fits in a stage");
  static constexpr size_t kSmem = static_cast<size_t>(kDecWarps) * kDecStages * kStage;
};

// Floats of one partial result: o [8 NT][D], m [8 NT], l [8 NT].
inline __host__ __device__ constexpr int dec_slot_floats(int D, int NT) { return 8 * NT * (D + 2); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// d += a (16 x 16) b (16 x 8), f16 or bf16 operands, fp32 sums.
template <bool kF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
// Two e4m3 codes -> two f16 values (exact).
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint16_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}
template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kF16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The length of sequence b, cut to what its page table can hold.
__device__ __forceinline__ int dec_len(const DecodeParams& p, int b, bool record) {
  const int64_t cap = static_cast<int64_t>(p.max_pages) * p.cache.page_size;
  const int n = __ldg(p.lens + b);
  if (n < 0 || n > cap) {
    if (record) record_error(kSiteBadIndex);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}

// Tiles of a sequence of len > 0 tokens (any: no sum here passes 2^31 - 1).
template <int kTile>
__device__ __forceinline__ int dec_tiles(int len) { return (len - 1) / kTile + 1; }

// N values of head h's output from their sum v and the weights' sum l (relative
// to the maximum m); l = 0 where no token counted.
template <int N>
__device__ __forceinline__ void dec_store(const DecodeParams& p, int b, int h, int d, const float (&v)[N], float m, float l) {
  const float r = l > 0.0f ? p.out_scale / l : l;      // NaN stays
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + b * p.o_token + h * p.o_head + d);
  if constexpr (N == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<false>(v[0] * r, v[1] * r), pack2<false>(v[2] * r, v[3] * r));
  else
    *dst = pack2<false>(v[0] * r, v[1] * r);
  if (p.lse && d == 0)
    p.lse[static_cast<int64_t>(b) * p.Hq + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Where a CTA is in the flat list: (sequence b, kv head and head block sub) and
// its tiles [j, j_end) that are this CTA's.
struct DecWalk {
  int b, sub, j, j_end;
  int len, n;          // the sequence's tokens and tiles
  int64_t start;       // of the item in the flat list
  bool done;
};

template <int D, bool kFp8, int kNT>
__global__ void __launch_bounds__(kDecThreads, kDecCtas) paged_decode_kernel(const DecodeParams p) {
  using Cfg = DecCfg<D, kFp8, kNT>;
  constexpr int kTok = Cfg::kTok, kTile = Cfg::kTile, kMT = D / 16, kKT = D / 16, kTT = kTok / 16;
  constexpr int kSlot = dec_slot_floats(D, kNT);
  constexpr float kWeight = kFp8 ? 32768.0f : 1.0f;       // what a weight of 1 is as an operand
  constexpr int kRowK = Cfg::kRowK, kRowV = Cfg::kRowV;
  constexpr uint64_t kFull = kTok == 64 ? ~0ull : (1ull << (kTok & 63)) - 1;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t s_scan[kDecThreads];
  __shared__ int64_t s_wsum[kDecWarps];
  __shared__ uint2 s_off[kDecWarps][kTok];                // a step's rows of k and v, in 16 bytes from the cache's base
  __shared__ uint64_t s_mask[kDecWarps][kDecStages];      // a step's tokens that count
  __shared__ float s_m[kDecWarps][8 * kNT], s_l[kDecWarps][8 * kNT];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * (kDecStages * Cfg::kStage);
  const int items = p.Hkv * p.blocks;

  grid_dependency_wait();

  // ---- the flat list: what lies before each thread's share of the sequences ----
  const int share = (p.B + kDecThreads - 1) / kDecThreads;
  const int b_lo = min(tid * share, p.B), b_hi = min(b_lo + share, p.B);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = dec_len(p, b, blockIdx.x == 0);
    if (len > 0) mine += dec_tiles<kTile>(len) + kDecItemCost;
  }
  mine *= items;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s_wsum[warp] = incl;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    if (w < warp) incl += s_wsum[w];
    total += s_wsum[w];
  }
  s_scan[tid] = incl - mine;
  __syncthreads();

  // sequences without tokens
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (dec_len(p, b, false) > 0) continue;
    for (int i = tid; i < p.Hq * (D / 8); i += kDecThreads)
      *reinterpret_cast<uint4*>(p.out + b * p.o_token + (i / (D / 8)) * p.o_head + (i % (D / 8)) * 8) =
          make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int h = tid; h < p.Hq; h += kDecThreads) p.lse[static_cast<int64_t>(b) * p.Hq + h] = -INFINITY;
  }

  const int64_t want = (total + kDecMinTiles - 1) / kDecMinTiles;
  const int64_t ctas = want < gridDim.x ? want : gridDim.x;
  // x / y; 64-bit divisions take hundreds of cycles, and few lists need them
  const bool narrow = (total + 1) * (ctas + 1) <= UINT32_MAX;
  auto quotient = [&](int64_t x, int64_t y) {
    return narrow ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y)) : x / y;
  };
  const int64_t t0 = blockIdx.x < ctas ? quotient(blockIdx.x * total, ctas) : 0;
  const int64_t t1 = blockIdx.x < ctas ? quotient((blockIdx.x + 1) * total, ctas) : 0;
  if (t0 >= t1) {
    grid_launch_dependents();
    return;
  }
  auto owner = [&](int64_t t) { return static_cast<int>(quotient((t + 1) * ctas - 1, total)); };

  auto enter = [&](DecWalk& w) {              // w.b, w.sub and w.start are set
    w.n = dec_tiles<kTile>(w.len);
    const int64_t first = w.start + kDecItemCost;
    w.j = t0 > first ? static_cast<int>(t0 - first) : 0;
    w.j_end = t1 - first < w.n ? static_cast<int>(t1 - first) : w.n;
    w.done = first >= t1;
  };
  auto next_item = [&](DecWalk& w) {
    w.start += w.n + kDecItemCost;
    if (w.start + kDecItemCost >= t1) {
      w.done = true;
      return;
    }
    if (++w.sub == items) {
      w.sub = 0;
      do {
        ++w.b;
        w.len = dec_len(p, w.b, false);
      } while (w.len == 0);
    }
    enter(w);
  };
  // the item of t0: the thread share it falls in, then along that share
  DecWalk cur;
  {
    int lo = 0, hi = kDecThreads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_scan[mid] <= t0) lo = mid;
      else hi = mid - 1;
    }
    int64_t at = s_scan[lo];
    int b = lo * share, per = 0;
    for (;; ++b) {
      cur.len = dec_len(p, b, false);
      per = cur.len > 0 ? dec_tiles<kTile>(cur.len) + kDecItemCost : 0;
      const int64_t here = static_cast<int64_t>(per) * items;
      if (t0 < at + here) break;
      at += here;
    }
    cur.b = b;
    cur.sub = static_cast<int>(quotient(t0 - at, per));
    cur.start = at + static_cast<int64_t>(cur.sub) * per;
    enter(cur);
    if (!cur.done && cur.j >= cur.j_end) cur.done = true;      // (t1 lies before its first tile)
  }
  if (cur.done) {
    grid_launch_dependents();
    return;
  }

  // ---- the copies of a step: page numbers one step ahead of the rows ----
  constexpr int kIds = (kTok + 31) / 32;      // rows per lane whose pages it looks up
  DecWalk pre = cur;                          // the next step to look up
  int id_page[kIds], id_at[kIds], id_head = 0, id_left = 0;
  auto look_up = [&]() {
    id_left = 0;
    if (pre.done) return;
    id_head = pre.sub / p.blocks;
    // (past the last token of a sequence of nearly 2^31 the first wraps, unused)
    const unsigned base = static_cast<unsigned>(pre.j) * kTile + warp * kTok;
    id_left = pre.len - pre.j * kTile - warp * kTok;
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const int r = lane + 32 * i;
      if (r < kTok && r < id_left) {
        const int tok = static_cast<int>(base + r);
        const int c = p.page_shift >= 0 ? tok >> p.page_shift : tok / p.cache.page_size;
        id_at[i] = tok - c * p.cache.page_size;
        id_page[i] = __ldg(p.table + pre.b * p.ld_table + c);
      }
    }
    if (++pre.j == pre.j_end) next_item(pre);
  };
  const int chunk = lane % Cfg::kChunks;
  const char* k_base = static_cast<const char*>(p.cache.k) + 16 * chunk;
  const char* v_base = static_cast<const char*>(p.cache.v) + 16 * chunk;
  const uint32_t k_dst = ring + (lane / Cfg::kChunks) * kRowK + 16 * chunk;
  const uint32_t v_dst = ring + kTok * kRowK + (lane / Cfg::kChunks) * kRowV + 16 * chunk;
  auto issue = [&](int stage) {
    constexpr int kUnit = kFp8 ? 16 : 8;       // elements in 16 bytes
    constexpr int kStep = 32 / Cfg::kChunks;   // rows per copy of the warp
    constexpr int kCopies = kTok / kStep;
    uint64_t mask = 0;
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const int r = lane + 32 * i;
      bool ok = r < kTok && r < id_left;
      if (ok && static_cast<unsigned>(id_page[i]) >= static_cast<uint64_t>(p.cache.num_pages)) {
        record_error(kSiteBadIndex);
        ok = false;
      }
      if (r < kTok) {
        uint2 off = make_uint2(0, 0);
        if (ok) {
          off.x = static_cast<uint32_t>((id_page[i] * p.cache.k_page + id_at[i] * p.cache.k_slot + id_head * p.cache.k_head) / kUnit);
          off.y = static_cast<uint32_t>((id_page[i] * p.cache.v_page + id_at[i] * p.cache.v_slot + id_head * p.cache.v_head) / kUnit);
        }
        s_off[warp][r] = off;
      }
      mask |= static_cast<uint64_t>(__ballot_sync(0xffffffffu, ok)) << (32 * i);
    }
    if (lane == 0) s_mask[warp][stage] = mask;
    __syncwarp();
    const uint2* off = &s_off[warp][lane / Cfg::kChunks];
    const uint32_t at = stage * Cfg::kStage;
    if (mask == kFull) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const uint2 x = off[i * kStep];
        cp_async16(k_dst + at + i * kStep * kRowK, k_base + static_cast<uint64_t>(x.x) * 16);
        cp_async16(v_dst + at + i * kStep * kRowV, v_base + static_cast<uint64_t>(x.y) * 16);
      }
    } else if (mask) {
      // rows that do not count are filled with zeros
#pragma unroll 1
      for (int i = 0; i < kCopies; ++i) {
        const uint2 x = off[i * kStep];
        const uint32_t n = (mask >> (lane / Cfg::kChunks + i * kStep)) & 1 ? 16 : 0;
        cp_async16_or_zero(k_dst + at + i * kStep * kRowK, k_base + static_cast<uint64_t>(x.x) * 16, n);
        cp_async16_or_zero(v_dst + at + i * kStep * kRowV, v_base + static_cast<uint64_t>(x.y) * 16, n);
      }
    }
    cp_async_commit();
  };

  look_up();
#pragma unroll
  for (int s = 0; s < kDecStages - 1; ++s) {
    issue(s);
    __syncwarp();                              // the offsets are read before the next ones
    look_up();
  }

  // q as it lies: lane (g, t4) reads the values of head g that it will hold
  constexpr int kRaw = 2 * kKT;
  uint32_t raw[kNT][kRaw];
  auto fetch_q = [&](const DecWalk& w) {
    const int hk = w.sub / p.blocks, hb = w.sub - hk * p.blocks;
    const int h0 = hk * p.group + hb * 8 * kNT;
    const int heads = min(8 * kNT, p.group - hb * 8 * kNT);
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int h = 8 * nt + g;
      const __nv_bfloat16* src = p.q + w.b * p.q_token + (h0 + h) * p.q_head;
      const bool ok = h < heads;
#pragma unroll
      for (int k = 0; k < kKT; ++k) {
        if constexpr (!kFp8) {
          raw[nt][2 * k] = ok ? __ldg(reinterpret_cast<const unsigned int*>(src + 16 * k + 2 * t4)) : 0u;
          raw[nt][2 * k + 1] = ok ? __ldg(reinterpret_cast<const unsigned int*>(src + 16 * k + 8 + 2 * t4)) : 0u;
        } else {
          const uint2 x = ok ? __ldg(reinterpret_cast<const uint2*>(src + 16 * (t4 + 4 * (k / 4)) + 4 * (k % 4))) : make_uint2(0, 0);
          raw[nt][2 * k] = x.x;
          raw[nt][2 * k + 1] = x.y;
        }
      }
    }
  };
  fetch_q(cur);

  int stage = 0;
  while (!cur.done) {
    const int hk = cur.sub / p.blocks, hb = cur.sub - hk * p.blocks;
    const int h0 = hk * p.group + hb * 8 * kNT;            // first query head
    const int heads = min(8 * kNT, p.group - hb * 8 * kNT);

    // q as the B operand.  bf16: as it lies.  e4m3 cache: f16, scaled by a
    // power of two so that a head's largest is in [2^14, 2^15): exact down to
    // 2^-28 of it, off by 2^-39 of it below.  k steps in the order of the k rows'
    // 16-byte chunks.
    uint32_t qf[kNT][kKT][2];
    float sc[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      if constexpr (!kFp8) {
#pragma unroll
        for (int k = 0; k < kKT; ++k) {
          qf[nt][k][0] = raw[nt][2 * k];
          qf[nt][k][1] = raw[nt][2 * k + 1];
        }
        sc[nt][0] = sc[nt][1] = p.scale_log2;
      } else {
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < kRaw; ++k) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(raw[nt][k])), fabsf(bf16_hi(raw[nt][k]))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^e <= amax < 2^(e+1); e from the exponent field, kept where 2^(14-e) and its
        // inverse are normal (126 for amax >= 2^127: at most 65280 then, in f16's range)
        const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -112), 126);
        const float down = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
#pragma unroll
        for (int k = 0; k < kKT; ++k) {
          qf[nt][k][0] = pack2<true>(bf16_lo(raw[nt][2 * k]) * down, bf16_hi(raw[nt][2 * k]) * down);
          qf[nt][k][1] = pack2<true>(bf16_lo(raw[nt][2 * k + 1]) * down, bf16_hi(raw[nt][2 * k + 1]) * down);
        }
        const float up = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
        sc[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t4);
        sc[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t4 + 4);
      }
    }
    float m[kNT][2], l[kNT][2], o[kNT][kMT][4];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kMT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }

    for (int j = cur.j; j < cur.j_end; ++j) {
      cp_async_wait<kDecStages - 2>();
      __syncwarp();
      {
        int ahead = stage + kDecStages - 1;    // the stage that the step before has left
        if (ahead >= kDecStages) ahead -= kDecStages;
        issue(ahead);
        look_up();
      }
      const uint32_t ka = ring + stage * Cfg::kStage, va = ka + kTok * kRowK;
      const uint64_t mask = s_mask[warp][stage];
      if (++stage == kDecStages) stage = 0;
      if (mask == 0) continue;
      // ---- scores: s[nt][tt]: tokens 16 tt + g (+8), heads 2 t4 (+1) ----
      float s[kNT][kTT][4];
#pragma unroll
      for (int tt = 0; tt < kTT; ++tt) {
        float s2[kNT][4];                      // two chains of products
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          s[nt][tt][0] = s[nt][tt][1] = s[nt][tt][2] = s[nt][tt][3] = 0.0f;
          s2[nt][0] = s2[nt][1] = s2[nt][2] = s2[nt][3] = 0.0f;
        }
        if constexpr (!kFp8) {
          const uint32_t at = ka + (16 * tt + (lane & 15)) * kRowK + (lane >> 4) * 16;
#pragma unroll
          for (int k = 0; k < kKT; ++k) {
            uint32_t a[4];
            ldsm4(a, at + 32 * k);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816<false>((k & 1) ? s2[nt] : s[nt][tt], a, qf[nt][k][0], qf[nt][k][1]);
          }
        } else {
          const uint32_t at = ka + (16 * tt + g) * kRowK + t4 * 16;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const uint4 r0 = lds128(at + 64 * c), r1 = lds128(at + 8 * kRowK + 64 * c);
            const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a[4] = {cvt_e4m3x2(static_cast<uint16_t>(w0[k])), cvt_e4m3x2(static_cast<uint16_t>(w1[k])),
                                     cvt_e4m3x2(static_cast<uint16_t>(w0[k] >> 16)),
                                     cvt_e4m3x2(static_cast<uint16_t>(w1[k] >> 16))};
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
                mma16816<true>((k & 1) ? s2[nt] : s[nt][tt], a, qf[nt][4 * c + k][0], qf[nt][4 * c + k][1]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][tt][i] = (s[nt][tt][i] + s2[nt][i]) * sc[nt][i & 1];
      }
      // ---- softmax ----
      if (mask != kFull) {
#pragma unroll
        for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            if (!((mask >> (16 * tt + g)) & 1)) s[nt][tt][0] = s[nt][tt][1] = -INFINITY;
            if (!((mask >> (16 * tt + g + 8)) & 1)) s[nt][tt][2] = s[nt][tt][3] = -INFINITY;
          }
      }
      uint32_t pf[kNT][kTT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < kTT; ++tt) {
          mx0 = fmaxf(mx0, fmaxf(s[nt][tt][0], s[nt][tt][2]));
          mx1 = fmaxf(mx1, fmaxf(s[nt][tt][1], s[nt][tt][3]));
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
        }
        if (__any_sync(0xffffffffu, mx0 > m[nt][0] || mx1 > m[nt][1])) {
          mx0 = fmaxf(mx0, m[nt][0]);
          mx1 = fmaxf(mx1, m[nt][1]);
          const float a0 = m[nt][0] == -INFINITY ? 0.0f : ex2(m[nt][0] - mx0);
          const float a1 = m[nt][1] == -INFINITY ? 0.0f : ex2(m[nt][1] - mx1);
          m[nt][0] = mx0;
          m[nt][1] = mx1;
          l[nt][0] *= a0;
          l[nt][1] *= a1;
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            o[nt][i][0] *= a0;
            o[nt][i][1] *= a1;
            o[nt][i][2] *= a0;
            o[nt][i][3] *= a1;
          }
        }
        // the weights meet v in 16 bits: bf16, each off by half an ulp at most; for
        // an e4m3 cache f16 (v is exact in it), times 2^15, so that they are off by half
        // an ulp down to 2^-29 of the maximum's and by 2^-40 of it below.  Their sum
        // l is of the unrounded.
        const float b0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
        for (int tt = 0; tt < kTT; ++tt) {
          const float p0 = ex2(s[nt][tt][0] - b0), p1 = ex2(s[nt][tt][1] - b1);
          const float p2 = ex2(s[nt][tt][2] - b0), p3 = ex2(s[nt][tt][3] - b1);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pf[nt][tt][0] = movmatrix_t(pack2<kFp8>(p0 * kWeight, p1 * kWeight));
          pf[nt][tt][1] = movmatrix_t(pack2<kFp8>(p2 * kWeight, p3 * kWeight));
        }
      }
      // ---- o^T += v^T p^T ----
#pragma unroll
      for (int tt = 0; tt < kTT; ++tt) {
        if constexpr (!kFp8) {
          const uint32_t at = va + (16 * tt + (lane & 7) + ((lane >> 4) << 3)) * kRowV + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            uint32_t a[4];
            ldsm4_t(a, at + 32 * i);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816<false>(o[nt][i], a, pf[nt][tt][0], pf[nt][tt][1]);
          }
        } else {
          // lane (g, t4) holds bytes g D/8 .. of tokens 2 t4, 2 t4 + 1, 2 t4 + 8,
          // 2 t4 + 9; row g of the i-th product is value g D/8 + 2 i, row g + 8 the next
          uint32_t w[4][D / 32];
          const uint32_t at = va + (16 * tt + 2 * t4) * kRowV + g * (D / 8);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t row = at + ((r & 1) + ((r >> 1) << 3)) * kRowV;
            if constexpr (D == 128) {
              const uint4 x = lds128(row);
              w[r][0] = x.x;
              w[r][1] = x.y;
              w[r][2] = x.z;
              w[r][3] = x.w;
            } else {
              const uint2 x = lds64(row);
              w[r][0] = x.x;
              w[r][1] = x.y;
            }
          }
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;     // bytes 2i, 2i + 1 of both tokens, paired by byte
            const uint32_t lo = __byte_perm(w[0][i >> 1], w[1][i >> 1], sel);
            const uint32_t hi = __byte_perm(w[2][i >> 1], w[3][i >> 1], sel);
            const uint32_t a[4] = {cvt_e4m3x2(static_cast<uint16_t>(lo)), cvt_e4m3x2(static_cast<uint16_t>(lo >> 16)),
                                   cvt_e4m3x2(static_cast<uint16_t>(hi)), cvt_e4m3x2(static_cast<uint16_t>(hi >> 16))};
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816<true>(o[nt][i], a, pf[nt][tt][0], pf[nt][tt][1]);
          }
        }
      }
    }

    // ---- the item's result: the four warps joined; each leaves its sums where
    // the rows of its last step were ----
    const int first = owner(cur.start + kDecItemCost), last = owner(cur.start + kDecItemCost + cur.n - 1);
    const bool whole = first == last;
    const int b = cur.b;
    float* slot = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (blockIdx.x == first ? 1 : 0)) * kSlot;
    next_item(cur);
    if (!cur.done) fetch_q(cur);               // arrives meanwhile
    const int used = stage == 0 ? kDecStages - 1 : stage - 1;
    auto sums = [&](int w) { return reinterpret_cast<float*>(smem + (w * kDecStages + used) * Cfg::kStage); };
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], x);
        l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], x);
      }
      const int h = 8 * nt + 2 * t4;                       // heads h, h + 1
      if (h < heads) {
        float* so = sums(warp) + h * Cfg::kPad;
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
          if constexpr (kFp8) {
            const int d = g * (D / 8) + 2 * i;
            constexpr float kBack = 1.0f / kWeight;
            *reinterpret_cast<float2*>(so + d) = make_float2(o[nt][i][0] * kBack, o[nt][i][2] * kBack);
            *reinterpret_cast<float2*>(so + Cfg::kPad + d) = make_float2(o[nt][i][1] * kBack, o[nt][i][3] * kBack);
          } else {
            const int d = 16 * i + g;
            so[d] = o[nt][i][0];
            so[d + 8] = o[nt][i][2];
            so[Cfg::kPad + d] = o[nt][i][1];
            so[Cfg::kPad + d + 8] = o[nt][i][3];
          }
        }
        if (g == 0) {
          s_m[warp][h] = m[nt][0];
          s_m[warp][h + 1] = m[nt][1];
          s_l[warp][h] = l[nt][0];
          s_l[warp][h + 1] = l[nt][1];
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < heads * (D / 4); i += kDecThreads) {
      const int h = i / (D / 4), d = (i % (D / 4)) * 4;
      float mm = s_m[0][h];
#pragma unroll
      for (int w = 1; w < kDecWarps; ++w) mm = fmaxf(mm, s_m[w][h]);
      float ll = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float a = s_m[w][h] == -INFINITY ? 0.0f : ex2(s_m[w][h] - mm);
        const float4 x = *reinterpret_cast<const float4*>(sums(w) + h * Cfg::kPad + d);
        ll += a * s_l[w][h];
        v.x += a * x.x;
        v.y += a * x.y;
        v.z += a * x.z;
        v.w += a * x.w;
      }
      if (whole) {
        const float o4[4] = {v.x, v.y, v.z, v.w};
        dec_store<4>(p, b, h0 + h, d, o4, mm, ll);
      } else {
        *reinterpret_cast<float4*>(slot + h * D + d) = v;
        if (d == 0) {
          slot[8 * kNT * D + h] = mm;
          slot[8 * kNT * (D + 1) + h] = ll;
        }
      }
    }
    __syncthreads();                           // the sums have been read
    if (!whole) {
      // (the barrier above puts the CTA's stores before
      // this release, and the one below puts its acquire before their loads)
      if (tid == 0) s_last = atomic_add_acq_rel_gpu(p.counters + first, 1) == last - first;
      __syncthreads();
      if (s_last) {
        // join the ranges' partial results in range order: a warp per head, its
        // lanes over the head's values
        if (tid == 0) p.counters[first] = 0;
        const int n = last - first + 1;
        auto part = [&](int i) {
          return p.partials + (static_cast<int64_t>(first + i) * 2 + (i == 0 ? 1 : 0)) * kSlot;
        };
        constexpr int kAhead = 8;
        constexpr int kPer = D / 32;             // values per lane
        for (int h0w = warp; h0w < heads; h0w += 2 * kDecWarps) {
          // two heads at a time, so that their loads run side by side
          float v[2][kPer] = {}, mm[2] = {-INFINITY, -INFINITY}, ll[2] = {};
          for (int i0 = 0; i0 < n; i0 += 32) {
            // lane i: range i0 + i; the first results on their way with the weights
            const int k = min(32, n - i0);
            float mi[2], li[2], x[2][kAhead][kPer];
            auto fetch = [&](int i) {
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const int h = h0w + z * kDecWarps;
                if (h >= heads) break;
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                  if (i + u < k) {
                    const float* src = part(i0 + i + u) + h * D + kPer * lane;
                    if constexpr (kPer == 4) {
                      const float4 y = __ldcg(reinterpret_cast<const float4*>(src));
                      x[z][u][0] = y.x;
                      x[z][u][1] = y.y;
                      x[z][u][2] = y.z;
                      x[z][u][3] = y.w;
                    } else {
                      const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
                      x[z][u][0] = y.x;
                      x[z][u][1] = y.y;
                    }
                  }
              }
            };
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int h = h0w + z * kDecWarps;
              const bool ok = lane < k && h < heads;
              mi[z] = ok ? __ldcg(part(i0 + lane) + 8 * kNT * D + h) : -INFINITY;
              li[z] = ok ? __ldcg(part(i0 + lane) + 8 * kNT * (D + 1) + h) : 0.0f;
            }
            fetch(0);
            float a[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              float mx = mi[z];
#pragma unroll
              for (int y = 16; y > 0; y >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
              mx = fmaxf(mx, mm[z]);
              const float old = mm[z] == -INFINITY ? 0.0f : ex2(mm[z] - mx);
              a[z] = mi[z] == -INFINITY ? 0.0f : ex2(mi[z] - mx);
              float sum = a[z] * li[z];
#pragma unroll
              for (int y = 16; y > 0; y >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
              ll[z] = ll[z] * old + sum;
              mm[z] = mx;
#pragma unroll
              for (int e = 0; e < kPer; ++e) v[z][e] *= old;
            }
            for (int i = 0; i < k; i += kAhead) {
              if (i > 0) fetch(i);
#pragma unroll
              for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                  const float f = __shfl_sync(0xffffffffu, a[z], (i + u) & 31);
                  if (i + u < k)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) v[z][e] = __fmaf_rn(f, x[z][u][e], v[z][e]);
                }
            }
          }
#pragma unroll
          for (int z = 0; z < 2; ++z)
            if (h0w + z * kDecWarps < heads) dec_store<kPer>(p, b, h0 + h0w + z * kDecWarps, kPer * lane, v[z], mm[z], ll[z]);
        }
      }
    }
  }
  cp_async_wait<0>();
  grid_launch_dependents();
}

}  // namespace fp8gq
