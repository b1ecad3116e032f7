// Attention over packed prompts on the 5th-generation tensor cores.
//
// Mathematics: per query row, one pass over the keys in tiles of 128 with the
// running maximum m and sum l of the softmax; O is rescaled when m moves.
//
// Bound: the tensor cores (4 D flops per visible pair and head) and, next to
// them, the exponentials: 128 x 128 of a tile take the MUFU as long as the
// tile's two products take the tensor core.  So a CTA carries two query tiles
// in turn: while one tile's scores are in the softmax, the other's products
// run.
//
// Query tile: 128 rows = R tokens x the G query heads of one kv head (R = 128 /
// G), loaded by one box [R][G][64] per half head, so that k and v are read once
// for the whole group, short prompts fill the tile, and a causal tile spans few
// tokens.  k and v tiles (128 tokens) go through a ring of shared-memory slots
// filled by TMA.  Scores and outputs live in TMEM (S0, S1, O0, O1); the weights
// P overwrite their scores as bf16 and are the A operand of the second product
// straight from TMEM; v is read as it lies (its N side contiguous).
//
// Warps 0-3 and 4-7: softmax, output (one thread per row of tile 0, 1).  Warp 8:
// TMA; it also clears the rows of the last v tile that lie past the sequence
// (another sequence's values, which a weight of 0 does not stop if they are
// NaN).  Warp 9: MMA.
#pragma once

#include "fp8gq_device.cuh"
#include "tensor_core.cuh"

namespace fp8gq {

struct PromptParams {
  __nv_bfloat16* out;
  float* lse;
  int64_t o_token, o_head;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, Tq, Tk, Hq, Hkv;
  int group, rows;          // query heads per kv head; tokens per query tile
  float scale_log2;         // |scale| log2(e)
  int negate;               // scale < 0
  int causal;
};

constexpr int kPrThreads = 384;
constexpr int kPrKeys = 128;          // keys per tile

template <int D>
struct PrCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * 128 * 128;        // bytes of a q, k or v tile
  static constexpr int kSlots = D == 128 ? 5 : 8;          // ring slots: k and v tiles in turn
  static constexpr size_t kSmem = 1024 + (2 + kSlots) * static_cast<size_t>(kTile);
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

// 32 columns of this warp's 32 lanes; the registers are valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : FP8GQ_R8(r, 0), FP8GQ_R8(r, 8), FP8GQ_R8(r, 16), FP8GQ_R8(r, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::FP8GQ_I8(r, 0),
      FP8GQ_I8(r, 8), FP8GQ_I8(r, 16), FP8GQ_I8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::FP8GQ_I8(r, 0),
      FP8GQ_I8(r, 8), "r"(addr)
      : "memory");
}
// Keeps the use of registers that tmem_ld32 fills behind tmem_wait_ld.
#define FP8GQ_B8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
__device__ __forceinline__ void tmem_loaded32(uint32_t* r) {
  asm volatile("" : FP8GQ_B8(r, 0), FP8GQ_B8(r, 8), FP8GQ_B8(r, 16), FP8GQ_B8(r, 24)::"memory");
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

// An offset cut to [0, hi]; one out of range is recorded.
__device__ __forceinline__ int pr_cut(int x, int hi) {
  if (x < 0 || x > hi) {
    record_error(kSiteBadIndex);
    return x < 0 ? 0 : hi;
  }
  return x;
}

// A CTA's work: two query tiles of one sequence and kv head.
struct PrWork {
  int q0, q1, k0, k1;       // the sequence's tokens
  int r0;                   // first token of the CTA within the sequence
  int n;                    // key tiles the last row sees
};

template <int D>
__global__ void __launch_bounds__(kPrThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap tq,
                                                                          const __grid_constant__ CUtensorMap tk,
                                                                          const __grid_constant__ CUtensorMap tv,
                                                                          const PromptParams p) {
  using Cfg = PrCfg<D>;
  constexpr int kSlots = Cfg::kSlots, kTile = Cfg::kTile;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t b_q, b_full[kSlots], b_free[kSlots], b_s[2], b_p[2], b_o, b_fix;
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[kPrThreads / 32];
  __shared__ PrWork s_work;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = base + 2 * kTile;

  if (warp == 8) {
    if (lane == 0) {
      prefetch_tensormap(&tq);
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
      mbar_init(&b_q, 1);
      for (int i = 0; i < kSlots; ++i) {
        mbar_init(&b_full[i], 1);
        mbar_init(&b_free[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&b_s[i], 1);
        mbar_init(&b_p[i], 128);
      }
      mbar_init(&b_o, 1);
      mbar_init(&b_fix, 32);
      fence_mbar_init();
    }
  } else if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_fence_before();
  }
  grid_dependency_wait();

  // ---- the work of this CTA: row blocks of the sequences in order, the last
  // (longest) of a sequence first ----
  const int hk = blockIdx.x % p.Hkv, tile = blockIdx.x / p.Hkv;
  const int span = 2 * p.rows;
  const int share = (p.B + kPrThreads - 1) / kPrThreads;
  const int b_lo = min(tid * share, p.B), b_hi = min(b_lo + share, p.B);
  auto tokens = [&](int b, int& q0, int& q1) {
    q0 = pr_cut(__ldg(p.cu_q + b), p.Tq);
    q1 = pr_cut(__ldg(p.cu_q + b + 1), p.Tq);
    if (q1 < q0) {
      record_error(kSiteBadIndex);
      q1 = q0;
    }
  };
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    int q0, q1;
    tokens(b, q0, q1);
    mine += (q1 - q0 + span - 1) / span;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s_scan[warp] = incl;
  if (tid == 0) s_work.q0 = -1;
  __syncthreads();
  for (int w = 0; w < warp; ++w) incl += s_scan[w];
  if (tile < incl && tile >= incl - mine) {
    int at = incl - mine;
    for (int b = b_lo; b < b_hi; ++b) {
      PrWork w;
      tokens(b, w.q0, w.q1);
      const int nb = (w.q1 - w.q0 + span - 1) / span;
      if (tile < at + nb) {
        w.k0 = pr_cut(__ldg(p.cu_k + b), p.Tk);
        w.k1 = pr_cut(__ldg(p.cu_k + b + 1), p.Tk);
        if (w.k1 < w.k0) {
          record_error(kSiteBadIndex);
          w.k1 = w.k0;
        }
        w.r0 = (nb - 1 - (tile - at)) * span;
        const int lq = w.q1 - w.q0, lk = w.k1 - w.k0;
        int seen = lk;
        if (p.causal) seen = min(lk, max(0, min(w.r0 + span, lq) + lk - lq));
        w.n = (seen + kPrKeys - 1) / kPrKeys;
        s_work = w;
        break;
      }
      at += nb;
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const PrWork w = s_work;
  const int lq = w.q1 - w.q0, lk = w.k1 - w.k0;
  const bool partial = w.n * kPrKeys > lk;       // the last tile reaches past the sequence
  bool ok = true;

  if (w.q0 >= 0) {
    if (warp == 8) {
      // ---- TMA ----
      if (lane == 0 && w.n > 0) {
        mbar_arrive_expect_tx(&b_q, 2 * Cfg::kHalves * p.group * p.rows * 128);
        for (int i = 0; i < 2; ++i)
          for (int h = 0; h < Cfg::kHalves; ++h)
            tma_load_3d(base + i * kTile + h * 16384, &tq, 64 * h, hk * p.group, w.q0 + w.r0 + i * p.rows, &b_q);
        int slot = 0, round = 0, issued = 0;
        for (int i = 0; i < 2 * w.n && ok; ++i) {      // k and v tiles in turn
          if (round > 0) ok = mbar_wait(&b_free[slot], (round - 1) & 1, kSitePrompt);
          if (!ok) break;
          mbar_arrive_expect_tx(&b_full[slot], kTile);
          for (int h = 0; h < Cfg::kHalves; ++h)
            tma_load_3d(ring + slot * kTile + h * 16384, (i & 1) ? &tv : &tk, 64 * h, hk, w.k0 + (i >> 1) * kPrKeys,
                        &b_full[slot]);
          ++issued;
          if (++slot == kSlots) {
            slot = 0;
            ++round;
          }
        }
        if (!ok) {
          // gave up: let the copies in flight land before the CTA may end
          mbar_wait(&b_q, 0, kSitePrompt);
          for (int i = issued > kSlots ? issued - kSlots : 0; i < issued; ++i)
            mbar_wait(&b_full[i % kSlots], (i / kSlots) & 1, kSitePrompt);
        }
      }
      // the last v tile's rows past the sequence: zeros
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (ok && w.n > 0 && partial) {
        const int i = 2 * w.n - 1, slot = i % kSlots;
        if (mbar_wait_warp(&b_full[slot], (i / kSlots) & 1, kSitePrompt, lane)) {
          const int valid = lk - (w.n - 1) * kPrKeys;
          const uint32_t v = ring + slot * kTile;
          for (int x = valid * 8 + lane; x < kPrKeys * 8; x += 32)
            for (int h = 0; h < Cfg::kHalves; ++h)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + h * 16384 + x * 16), "r"(0u) : "memory");
          fence_proxy_async_smem();
          mbar_arrive(&b_fix);
        }
      }
    } else if (warp == 9) {
      // ---- MMA ----
      if (lane == 0 && w.n > 0) {
        const uint32_t id_s = pr_idesc(kPrKeys, false, p.negate != 0), id_o = pr_idesc(D, true, false);
        int slot = 0, round = 0;
        auto next = [&]() {
          if (++slot == kSlots) {
            slot = 0;
            ++round;
          }
        };
        auto scores = [&](int i, int at) {
          const uint32_t a = base + i * kTile, b = ring + at * kTile;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tmem + i * 128, pr_desc(a + (k >> 2) * 16384 + (k & 3) * 32, 16), pr_desc(b + (k >> 2) * 16384 + (k & 3) * 32, 16),
                   id_s, k > 0);
          mma_commit(&b_s[i]);
        };
        auto values = [&](int i, int at, bool first) {
          const uint32_t b = ring + at * kTile;
#pragma unroll
          for (int k = 0; k < kPrKeys / 16; ++k)
            mma_ts(tmem + 256 + i * 128, tmem + i * 128 + 8 * k, pr_desc(b + k * 2048, 16384), id_o, !first || k > 0);
        };
        ok = mbar_wait(&b_q, 0, kSitePrompt) && mbar_wait(&b_full[0], 0, kSitePrompt);
        if (ok) {
          tc_fence_after();
          scores(0, 0);
          scores(1, 0);
          mma_commit(&b_free[0]);
          next();
        }
        for (int j = 0; j < w.n && ok; ++j) {
          const int v_slot = slot, v_round = round;
          ok = mbar_wait(&b_full[v_slot], v_round & 1, kSitePrompt);
          if (ok && j == w.n - 1 && partial) ok = mbar_wait(&b_fix, 0, kSitePrompt);
          next();
          const int k_slot = slot, k_round = round;
          for (int i = 0; i < 2 && ok; ++i) {
            ok = mbar_wait(&b_p[i], j & 1, kSitePrompt);
            if (!ok) break;
            tc_fence_after();
            values(i, v_slot, j == 0);
            if (j + 1 < w.n) {
              if (i == 0) ok = mbar_wait(&b_full[k_slot], k_round & 1, kSitePrompt);
              if (!ok) break;
              scores(i, k_slot);
            }
          }
          if (!ok) break;
          mma_commit(&b_free[v_slot]);
          if (j + 1 < w.n) {
            mma_commit(&b_free[k_slot]);
            next();
          }
        }
        mma_commit(&b_o);
      }
    } else if (warp < 8) {
      // ---- softmax and output: one thread per row ----
      const int i = warp >> 2, row = tid & 127;
      const int tok = w.r0 + i * p.rows + row / p.group;        // token within the sequence
      const int head = hk * p.group + row % p.group;
      const bool live = row < p.rows * p.group && tok < lq;
      int lim = lk;                                              // keys this row sees
      if (p.causal) lim = max(0, min(lk, tok + 1 + lk - lq));
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lane_base + i * 128, to = tmem + lane_base + 256 + i * 128;
      const float c = p.scale_log2;
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < w.n && ok; ++j) {
        ok = mbar_wait_warp(&b_s[i], j & 1, kSitePrompt, lane);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld32(ts + 32 * x, s + 32 * x);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_loaded32(s + 32 * x);
        const int vis = lim - j * kPrKeys;
        if (__any_sync(0xffffffffu, vis < kPrKeys)) {
#pragma unroll
          for (int x = 0; x < 128; ++x)
            if (x >= vis) s[x] = 0xff800000u;
        }
        float mx = __uint_as_float(s[0]);
#pragma unroll
        for (int x = 1; x < 128; ++x) mx = fmaxf(mx, __uint_as_float(s[x]));
        // O keeps its reference maximum until a row's grows by more than 2^8
        const bool move = (mx - m) * c > 8.0f || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float mn = fmaxf(m, mx);
          if (j > 0) {
            const float a = m == -INFINITY ? 0.0f : ex2f((m - mn) * c);
            l *= a;
            // (O of the tiles so far is complete: its products were issued before these scores)
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
              uint32_t o[32];
              tmem_ld32(to + x, o);
              tmem_wait_ld();
              tmem_loaded32(o);
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * a);
              tmem_st32(to + x, o);
            }
          }
          m = mn;
        }
        const float mc = m == -INFINITY ? 0.0f : m * c;
        // weights in bf16 (half an ulp each, in [0, 2^8]); l sums the unrounded
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int x = 0; x < 128; x += 32) {
          uint32_t q[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const float a = ex2f(__fmaf_rn(__uint_as_float(s[x + 2 * y]), c, -mc));
            const float b = ex2f(__fmaf_rn(__uint_as_float(s[x + 2 * y + 1]), c, -mc));
            sum0 += a;
            sum1 += b;
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            q[y] = *reinterpret_cast<const uint32_t*>(&h);
          }
          tmem_st16(ts + x / 2, q);
        }
        l += sum0 + sum1;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&b_p[i]);
      }
      if (w.n > 0) ok = mbar_wait_warp(&b_o, 0, kSitePrompt, lane) && ok;
      tc_fence_after();
      const float r = l > 0.0f ? 1.0f / l : l;                   // a row that sees nothing: 0; NaN stays
      __nv_bfloat16* dst = p.out + (static_cast<int64_t>(w.q0) + tok) * p.o_token + head * p.o_head;
#pragma unroll 1
      for (int x = 0; x < D; x += 32) {
        uint32_t o[32];
        if (w.n > 0) {
          tmem_ld32(to + x, o);
          tmem_wait_ld();
          tmem_loaded32(o);
        }
        if (live) {
#pragma unroll
          for (int y = 0; y < 32; y += 8) {
            float v[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) v[z] = l == 0.0f ? 0.0f : __uint_as_float(o[y + z]) * r;
            uint4 h;
            uint32_t* hw = reinterpret_cast<uint32_t*>(&h);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * z], v[2 * z + 1]);
              hw[z] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(dst + x + y) = h;
          }
        }
      }
      if (live && p.lse)
        p.lse[(static_cast<int64_t>(w.q0) + tok) * p.Hq + head] =
            l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m * c) + log2f(l)) * 0.6931471805599453f;
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
