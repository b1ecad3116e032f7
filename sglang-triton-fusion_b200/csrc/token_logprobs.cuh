// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits.
//
// Mathematics: in units of log 2, with r = log2(e) max x (rounded: any reference
// near the maximum will do), y = log2(e) x - r in one fma, s = sum 2^y and
// e = sum 2^y y:  logprob(t) = ln 2 (y_t - log2 s), entropy = ln 2 (log2 s - e / s).
// Each thread keeps (r, s, e) of what it has read, rescaled when r moves; such
// triples join in any grouping.
//
// Bound: HBM, one pass, streamed through a ring of bulk copies; next to it the exponentials (one MUFU operation per
// value, 16 a cycle and SM: 72 % of the time that a bf16 row takes to arrive),
// so the rest is kept to packed pairs: clamp, fma, add, fma.
//
// A row is read by a cluster of 1 to 16 CTAs (more for fewer rows), joined over
// distributed shared memory: one launch, no scratch.  The alternatives cost
// the stream nothing: each thread keeps the maximum of each quarter of what it
// reads (a column).  The top_k-th largest of the CTA's 256 threads' maxima is a
// lower bound of its top_k-th value that few values pass, and they all lie in
// the columns whose maximum passes it; only those are read again, by all
// threads, and ranked.  Inserting candidates into sorted lists as they stream by
// was measured 38 us slower at 2048 x 151936 bf16 with 8 alternatives.  Sums
// join in a fixed order and candidates are ranked by value and index, so
// results do not depend on timing.
//
// Measured in a CUDA graph, 151936 logits a row: 2048 rows bf16 119 us (5.2 TB/s;
// MUFU 66 % and issue 72 % busy), 37 rows fp32 13.1 to 13.6 us, 1 row bf16 8.2 to 8.8
// us (latency).
#pragma once

#include "fp8gq_device.cuh"
#include "tensor_core.cuh"

namespace fp8gq {

constexpr int kMaxTop = 32;
constexpr int kLpWarps = 8;
constexpr int kLpThreads = 32 * kLpWarps;
constexpr int kLpUnroll = 4;              // 16-byte vectors per lane and chunk (32 bf16 or 16 fp32 values)
constexpr int kLpParts = 4;               // columns per thread: what it reads in this many parts
constexpr int kLpPool = 512;              // candidates of a CTA
constexpr int kLpStages = 3;              // steps of the CTA (16 KB) in flight
constexpr int kLpStepBytes = kLpThreads * kLpUnroll * 16;

struct LogprobParams {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int T, V, K;
  int cluster;
};

using lp_key = unsigned long long;

// A logit and its index as one key: larger logits first, equal ones (0 and -0
// too) by ascending index; NaN above +inf.  0 is below every key.
__device__ __forceinline__ lp_key logit_key(float x, int i) {
  uint32_t b = x != x ? 0x7fffffffu : __float_as_uint(x + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<lp_key>(b) << 32) | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ float key_logit(lp_key key) {
  uint32_t b = static_cast<uint32_t>(key >> 32);
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int key_index(lp_key key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// Order-preserving integer of a float (no NaN; -0 as 0), and the largest float
// below the one of an order.
__device__ __forceinline__ int float_order(float x) {
  const int b = __float_as_int(x + 0.0f);
  return b < 0 ? b ^ 0x7fffffff : b;
}
constexpr int kOrderMinusInf = static_cast<int>(0xff800000u ^ 0x7fffffffu);
__device__ __forceinline__ float just_below(int order) {
  const int o = order <= kOrderMinusInf ? kOrderMinusInf : order == 0 ? -2 : order - 1;   // -1 would be -0
  return __int_as_float(o < 0 ? o ^ 0x7fffffff : o);
}

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int64_t i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(row[i]);
  else return row[i];
}

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The sums see values clamped to -1e37, so that y stays finite for -inf and for
// the lowest finite values; the clamp keeps NaN.  A row is regular while its
// maximum is below 1e6 in size, so that the rounding of r (2^-24 of it, the y of
// the maximum) stays small and a clamped value weighs nothing; any other is
// done again by lp_irregular.
constexpr float kLpLowest = -1e37f;
constexpr float kLpFloor = -2e6f;         // r of nothing yet: below every regular row's
__device__ __forceinline__ bool lp_regular(float r, float s) { return fabsf(r) < 1e6f && s == s; }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {      // bf16 pairs, NaN ignored
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct LpSums {
  float m, s, e;      // r, s, e above
};
__device__ __forceinline__ float lp_shift(float from, float to) { return fmaxf(from - to, -2000.0f); }
__device__ __forceinline__ void lp_move(LpSums& a, float m) {
  const float d = lp_shift(a.m, m), f = lp_ex2(d);
  a.e = (a.e + d * a.s) * f;
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void lp_join(LpSums& a, LpSums b) {
  const float m = fmaxf(a.m, b.m);
  lp_move(a, m);
  lp_move(b, m);
  a.s += b.s;
  a.e += b.e;
}
__device__ __forceinline__ LpSums lp_shfl_xor(const LpSums& a, int x) {
  return {__shfl_xor_sync(0xffffffffu, a.m, x), __shfl_xor_sync(0xffffffffu, a.s, x), __shfl_xor_sync(0xffffffffu, a.e, x)};
}

// The sums of n lanes (a power of two) joined, on every lane; both lanes of a
// pair join in the same order.
__device__ __forceinline__ LpSums lp_join_lanes(LpSums a, int n, int lane) {
  for (int x = 1; x < n; x <<= 1) {
    LpSums o = lp_shfl_xor(a, x);
    if (lane & x) {
      lp_join(o, a);
      a = o;
    } else {
      lp_join(a, o);
    }
  }
  return a;
}

// A chunk of a lane: kLpUnroll 16-byte vectors.
template <typename T>
struct LpChunk {
  uint32_t w[4 * kLpUnroll];
  // from shared memory; `left` vectors of the CTA's step are there
  __device__ __forceinline__ void load(uint32_t step, int v, int left) {
    constexpr uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;      // -inf
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      uint4 a = make_uint4(none, none, none, none);
      if (v + 32 * u < left)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w)
                     : "r"(step + 16 * (v + 32 * u)) : "memory");
      w[4 * u] = a.x;
      w[4 * u + 1] = a.y;
      w[4 * u + 2] = a.z;
      w[4 * u + 3] = a.w;
    }
  }
  __device__ __forceinline__ float max() const {
    if constexpr (sizeof(T) == 2) {
      uint32_t m = w[0];
#pragma unroll
      for (int i = 1; i < 4 * kLpUnroll; ++i) m = max2(m, w[i]);
      return fmaxf(fmaxf(bf16_lo(m), bf16_hi(m)), -INFINITY);
    } else {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * kLpUnroll; ++i) m = fmaxf(m, __uint_as_float(w[i]));
      return m;
    }
  }
  // s and e in two halves each (the packed operations' lanes)
  __device__ __forceinline__ void add(float r, float2& s, float2& e) const {
    const float2 l2 = make_float2(kLog2e, kLog2e), nr = make_float2(-r, -r);
#pragma unroll
    for (int i = 0; i < 4 * kLpUnroll; i += sizeof(T) == 2 ? 1 : 2) {
      float2 x;
      if constexpr (sizeof(T) == 2) {
        const uint32_t c = max2_nan(w[i], 0xfcf1fcf1u);      // -1e37 as bf16
        x = make_float2(bf16_lo(c), bf16_hi(c));
      } else {
        x = make_float2(max_nan(__uint_as_float(w[i]), kLpLowest), max_nan(__uint_as_float(w[i + 1]), kLpLowest));
      }
      const float2 y = fma2(x, l2, nr);
      const float2 f = make_float2(lp_ex2(y.x), lp_ex2(y.y));
      s = add2(s, f);
      e = fma2(f, y, e);
    }
  }
};

// Two lists in descending order across the lanes -> the best 32 of both.
__device__ __forceinline__ lp_key lp_merge(lp_key a, lp_key b, int lane) {
  const lp_key r = __shfl_sync(0xffffffffu, b, 31 - lane);
  a = a > r ? a : r;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    const lp_key o = __shfl_xor_sync(0xffffffffu, a, x);
    const bool up = (lane & x) == 0;
    a = (up == (a > o)) ? a : o;
  }
  return a;
}

// The lanes' values (no NaN) in descending order.
__device__ __forceinline__ float lp_sort_lanes(float v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int x = k >> 1; x > 0; x >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, x);
      const bool keep_max = ((lane & x) == 0) == ((lane & k) == 0);
      v = keep_max ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

// The K-th largest of the CTA's values.
__device__ __forceinline__ float lp_kth(float v, int K, float (*lists)[32], int warp, int lane) {
  v = lp_sort_lanes(v, lane);
  lists[warp][lane] = v;
#pragma unroll
  for (int n = kLpWarps / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (warp < n) {
      v = fmaxf(v, lists[warp + n][31 - lane]);      // descending and ascending: the best 32, bitonic
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, x);
        v = (lane & x) == 0 ? fmaxf(v, o) : fminf(v, o);
      }
      lists[warp][lane] = v;
    }
  }
  __syncthreads();
  return lists[0][K - 1];
}

// The CTA's 8 lists in shared memory -> the best 32, on warp 0's lanes.
__device__ __forceinline__ lp_key lp_merge_lists(lp_key (*lists)[32], int warp, int lane) {
#pragma unroll
  for (int n = kLpWarps / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (warp < n) lists[warp][lane] = lp_merge(lists[warp][lane], lists[warp + n][lane], lane);
  }
  return lists[0][lane];      // warp 0 wrote it itself
}

// Keeps a value that passes the threshold.
__device__ __forceinline__ void lp_keep(float x, int id, float low, int* found, lp_key* pool) {
  if (x > low) {
    const int at = atomicAdd(found, 1);
    if (at < kLpPool) pool[at] = logit_key(x, id);
  }
}

// The largest of the CTA's keys, on every thread.
__device__ __forceinline__ lp_key lp_block_max(lp_key best, lp_key* scratch, int warp, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const lp_key x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
  }
  __syncthreads();
  if (lane == 0) scratch[warp] = best;
  __syncthreads();
  for (int w = 0; w < kLpWarps; ++w) best = scratch[w] > best ? scratch[w] : best;
  return best;
}

// The top_k largest keys of row[lo, hi), row[0, head) and row[tail, V), one pass
// each: where more values pass the threshold than the pool holds (long runs of
// equal logits, or few columns with any above -inf).
template <typename T>
__device__ __noinline__ void lp_by_passes(const T* row, int lo, int hi, int head, int tail, int V, int K, lp_key* out,
                                          lp_key* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int body = hi - lo, n = body + head + (V - tail);
  lp_key last = ~0ull;
  for (int k = 0; k < K && last; ++k) {
    lp_key best = 0;
    for (int i = tid; i < n; i += kLpThreads) {
      const int id = i < body ? lo + i : i < body + head ? i - body : tail + i - body - head;
      const float x = logit_at(row, id);
      const lp_key key = logit_key(x, id);
      if (x > -INFINITY && key < last && key > best) best = key;
    }
    last = lp_block_max(best, scratch, warp, lane);
    if (tid == 0) out[k] = last;
  }
  __syncthreads();
}

// A row with NaN, infinite or very large values, or none above -inf, by one
// CTA: a pass for the maximum, one for the sums, one per alternative.
template <typename T>
__device__ __noinline__ void lp_irregular(const LogprobParams& p, const T* row, int t, lp_key* keys, LpSums* sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < p.V; i += kLpThreads) {
    const float x = logit_at(row, i);
    nan |= x != x;
    m = fmaxf(m, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  nan = __syncthreads_or(nan) != 0;
  if (lane == 0) sums[warp].m = m;
  __syncthreads();
  for (int w = 0; w < kLpWarps; ++w) m = fmaxf(m, sums[w].m);
  nan |= isinf(m);
  float s = 0.0f, e = 0.0f;
  for (int i = tid; i < p.V; i += kLpThreads) {
    const float y = logit_at(row, i) - m, f = expf(y);
    s += f;
    if (f > 0.0f) e += f * y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
  }
  if (lane == 0) {
    sums[warp].s = s;
    sums[warp].e = e;
  }
  __syncthreads();
  s = e = 0.0f;
  for (int w = 0; w < kLpWarps; ++w) {
    s += sums[w].s;
    e += sums[w].e;
  }
  const float ls = nan ? NAN : logf(s);
  if (tid == 0) {
    if (p.logprobs) {
      const int64_t tok = p.tokens[t];
      if (tok >= p.V) record_error(kSiteBadIndex);
      p.logprobs[t] = tok < 0 ? 0.0f : tok >= p.V ? NAN : (logit_at(row, tok) - m) - ls;
    }
    if (p.entropy) p.entropy[t] = ls - e / s;
  }
  lp_key last = ~0ull;
  for (int k = 0; k < p.K; ++k) {
    lp_key best = 0;
    for (int i = tid; i < p.V; i += kLpThreads) {
      const lp_key x = logit_key(logit_at(row, i), i);
      if (x < last && x > best) best = x;
    }
    last = lp_block_max(best, keys, warp, lane);
    if (tid == 0) {
      p.top_ids[static_cast<int64_t>(t) * p.K + k] = key_index(last);
      p.top_logprobs[static_cast<int64_t>(t) * p.K + k] = (key_logit(last) - m) - ls;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobParams p) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kStep = kLpThreads * kLpUnroll;
  extern __shared__ __align__(128) unsigned char ring[];      // the stream's steps; the candidates once it has ended
  struct Found {
    lp_key pool[kLpPool];
    lp_key list[kLpWarps][32];
    float max[kLpWarps][32];
    uint16_t column[kLpParts * kLpThreads];
  };
  static_assert(sizeof(Found) <= kLpStages * kLpStepBytes, "the candidates fit the ring");
  Found& found = *reinterpret_cast<Found*>(ring);
  __shared__ uint64_t s_full[kLpStages], s_free[kLpStages];
  __shared__ lp_key s_out[32];                   // this CTA's best, read by the cluster
  __shared__ float s_part[kLpParts][kLpThreads];
  __shared__ LpSums s_sum[kLpWarps], s_total;
  __shared__ int s_columns, s_found, s_regular;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int t = blockIdx.x / p.cluster;
  const int K = p.K;
  if (tid == 0) s_columns = s_found = 0;         // used after the barriers of lp_kth
  if (tid < 32) s_out[tid] = 0;
  if (tid == 0) {
    for (int i = 0; i < kLpStages; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kLpWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  grid_dependency_wait();

  // a row: up to kVec - 1 values before the first 16-byte boundary, vectors, up to kVec - 1 after
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  const int before = min(p.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (p.V - before) / kVec;
  const int after = before + vectors * kVec;
  const uint4* vec = reinterpret_cast<const uint4*>(row + before);
  const int v_lo = static_cast<int>(static_cast<int64_t>(vectors) * rank / p.cluster);
  const int v_hi = static_cast<int>(static_cast<int64_t>(vectors) * (rank + 1) / p.cluster);

  // the stream
  LpSums sum = {kLpFloor, 0.0f, 0.0f};
  float2 s2 = make_float2(0.0f, 0.0f), e2 = make_float2(0.0f, 0.0f);
  const int its = (v_hi - v_lo + kStep - 1) / kStep, part_its = (its + kLpParts - 1) / kLpParts;
  float most = -INFINITY, part = -INFINITY;
  int it = 0, parts = 0;
  const uint64_t policy = l2_policy_evict_first();
  auto copy = [&](int i, int stage) {            // step i of this CTA
    const int n = min(kStep, v_hi - v_lo - i * kStep);
    mbar_arrive_expect_tx(&s_full[stage], 16 * n);
    bulk_g2s(ring + stage * kLpStepBytes, vec + v_lo + i * kStep, 16 * n, &s_full[stage], policy);
  };
  bool ok = true;
  int sent = 0;                                  // thread 0: steps on their way or there
  if (tid == 0)
    for (; sent < min(kLpStages, its); ++sent) copy(sent, sent);
  // the given token's logit, fetched meanwhile
  int64_t token = -1;
  float token_logit = 0.0f;
  if (tid == 0 && rank == 0 && p.logprobs) {
    token = p.tokens[t];
    if (token >= p.V) record_error(kSiteBadIndex);
    else if (token >= 0) token_logit = logit_at(row, token);
  }
  int stage = 0;
  uint32_t phase = 0;
  for (int i = 0; i < its; ++i) {
    LpChunk<T> now;
    ok = mbar_wait_warp(&s_full[stage], phase, kSiteScore, lane);
    if (!ok) break;
    now.load(smem_u32(ring) + stage * kLpStepBytes, warp * 32 * kLpUnroll + lane, v_hi - v_lo - i * kStep);
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_free[stage]);
    // the stage of the step before, which every warp has read by now or soon (unless
    // one gave up: then nothing more is sent)
    if (tid == 0 && i > 0 && sent == i - 1 + kLpStages && sent < its) {
      const int before_stage = stage == 0 ? kLpStages - 1 : stage - 1;
      if (mbar_wait(&s_free[before_stage], stage == 0 ? phase ^ 1 : phase, kSiteScore)) copy(sent++, before_stage);
    }
    if (++stage == kLpStages) {
      stage = 0;
      phase ^= 1;
    }
    const float mx = now.max();
    part = fmaxf(part, mx);
    if (++it == part_its) {
      s_part[parts++][tid] = part;
      most = fmaxf(most, part);
      part = -INFINITY;
      it = 0;
    }
    const float r = mx * kLog2e;
    if (r > sum.m) {
      const float d = lp_shift(sum.m, r), f = lp_ex2(d);
      e2 = fma2(s2, make_float2(d, d), e2);
      e2 = make_float2(e2.x * f, e2.y * f);
      s2 = make_float2(s2.x * f, s2.y * f);
      sum.m = r;
    }
    now.add(sum.m, s2, e2);
  }
  if (it > 0) {
    s_part[parts++][tid] = part;
    most = fmaxf(most, part);
  }
  sum.s = s2.x + s2.y;
  sum.e = e2.x + e2.y;

  // where a wait gave up, the copies sent land before the ring takes the candidates
  // or goes to another CTA, and the row is done again as an irregular one
  const bool gave_up = __syncthreads_or(!ok) != 0;           // (the ring has been read)
  if (gave_up) {
    if (tid == 0)
      for (int i = max(sent - kLpStages, 0); i < sent; ++i) mbar_wait(&s_full[i % kLpStages], (i / kLpStages) & 1, kSiteScore);
    sum.s = NAN;
    __syncthreads();
  }

  // the candidates
  float low = -INFINITY;
  if (K > 0 && !gave_up) {
    low = just_below(float_order(lp_kth(most, K, found.max, warp, lane)));
    // the columns to read again, listed (in any order)
    unsigned is[kLpParts];
    int here = 0;
#pragma unroll
    for (int i = 0; i < kLpParts; ++i) {
      is[i] = __ballot_sync(0xffffffffu, i < parts && s_part[i][tid] > low);
      here += __popc(is[i]);
    }
    if (here) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&s_columns, here);
      at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
      for (int i = 0; i < kLpParts; ++i) {
        if ((is[i] >> lane) & 1)
          found.column[at + __popc(is[i] & ((1u << lane) - 1))] = static_cast<uint16_t>(i * kLpThreads + tid);
        at += __popc(is[i]);
      }
    }
    __syncthreads();
    // their vectors, spread over the CTA's threads
    const int deep = kLpUnroll * part_its;       // vectors of a column, at most
    const int again = s_columns * deep;
    for (int f = tid; f < again; f += kLpThreads) {
      const int col = f / deep, c = found.column[col] % kLpThreads;
      const int j = f - col * deep + deep * (found.column[col] / kLpThreads);
      const int v = v_lo + (c & ~31) * kLpUnroll + (c & 31) + 32 * (j % kLpUnroll) + kStep * (j / kLpUnroll);
      if (v < v_hi) {
        const uint4 a = __ldcg(vec + v);
        const T* x = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < kVec; ++i) lp_keep(logit_at(x, i), before + v * kVec + i, low, &s_found, found.pool);
      }
    }
  }
  // the values outside the vectors: one per lane of one warp
  if (warp == 0 && rank == 0) {
    const int id = lane < 8 ? lane : after + lane - 8;
    const float x = (lane < 8 ? lane < before : id < p.V && lane < 16) ? logit_at(row, id) : -INFINITY;
    const float c = max_nan(x, kLpLowest);
    if (c * kLog2e > sum.m) lp_move(sum, c * kLog2e);
    const float y = __fmaf_rn(c, kLog2e, -sum.m), f = lp_ex2(y);
    sum.s += f;
    sum.e = __fmaf_rn(f, y, sum.e);
    if (K > 0) lp_keep(x, id, low, &s_found, found.pool);
  }

  // the warps, in order
  sum = lp_join_lanes(sum, 32, lane);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (K > 0) {
    const int n = s_found;
    if (n <= kLpPool) {
      // a candidate's place: how many are above it
      for (int i = tid; i < n; i += kLpThreads) {
        const lp_key x = found.pool[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += found.pool[j] > x;
        if (above < K) s_out[above] = x;
      }
    } else {
      __syncthreads();
      lp_by_passes(row, before + v_lo * kVec, before + v_hi * kVec, rank == 0 ? before : 0, rank == 0 ? after : p.V, p.V,
                   K, s_out, found.pool);
    }
  }
  if (warp == 0) {
    sum = lp_join_lanes(s_sum[lane % kLpWarps], kLpWarps, lane);
    if (lane == 0) s_total = sum;
  }

  // the cluster's CTAs, in order, by the first
  lp_key key = 0;
  if (p.cluster > 1) {
    cluster_sync_all();
    if (rank == 0) {
      if (K > 0) {
        lp_key a = 0, b = 0;
        if (warp < p.cluster) {
          const uint32_t at = dsmem_addr(&s_out[lane], warp);
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(a) : "r"(at) : "memory");
        }
        if (warp + kLpWarps < p.cluster) {
          const uint32_t at = dsmem_addr(&s_out[lane], warp + kLpWarps);
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(b) : "r"(at) : "memory");
          a = lp_merge(a, b, lane);
        }
        found.list[warp][lane] = a;
        key = lp_merge_lists(found.list, warp, lane);
      }
      if (warp == 0) {
        LpSums o = {kLpFloor, 0.0f, 0.0f};
        if (lane < p.cluster) {
          o.m = ld_dsmem(dsmem_addr(&s_total.m, lane));
          o.s = ld_dsmem(dsmem_addr(&s_total.s, lane));
          o.e = ld_dsmem(dsmem_addr(&s_total.e, lane));
        }
        sum = lp_join_lanes(o, 16, lane);
      }
    }
    cluster_sync_all();                          // the others' shared memory has been read
    if (rank != 0) {
      grid_launch_dependents();
      return;
    }
  } else {
    __syncthreads();
    key = s_out[lane];
  }

  // results: warp 0 for a regular row
  if (warp == 0) {
    sum.m = __shfl_sync(0xffffffffu, sum.m, 0);
    sum.s = __shfl_sync(0xffffffffu, sum.s, 0);
    sum.e = __shfl_sync(0xffffffffu, sum.e, 0);
    const bool regular = lp_regular(sum.m, sum.s);
    if (lane == 0) s_regular = regular;
    if (regular) {
      const float l2s = log2f(sum.s);
      // x log2(e) of a value near the type's lowest (a mask) is past fp32 where x is
      // not; next to such an x the roundings of r do not show
      auto logprob = [&](float x) {
        return x < kLpLowest ? x - kLn2 * (sum.m + l2s) : kLn2 * (__fmaf_rn(x, kLog2e, -sum.m) - l2s);
      };
      if (lane == 0) {
        if (p.logprobs) p.logprobs[t] = token < 0 ? 0.0f : token >= p.V ? NAN : logprob(token_logit);
        if (p.entropy) p.entropy[t] = kLn2 * (l2s - sum.e / sum.s);
      }
      if (K > 0) {
        // fewer than K tokens above -inf: the first of the others follow, which
        // are among the first K
        const int n = __popc(__ballot_sync(0xffffffffu, key != 0 && lane < K));
        if (n < K) {
          bool in = false;
          for (int i = 0; i < n; ++i) in |= key_index(__shfl_sync(0xffffffffu, key, i)) == lane;
          unsigned f = __ballot_sync(0xffffffffu, !in && lane < K);
          for (int i = n; i < lane; ++i) f &= f - 1;             // entry n + i: the i-th of them
          if (lane >= n && lane < K) key = logit_key(-INFINITY, __ffs(f) - 1);
        }
        if (lane < K) {
          p.top_ids[static_cast<int64_t>(t) * K + lane] = key_index(key);
          p.top_logprobs[static_cast<int64_t>(t) * K + lane] = logprob(key_logit(key));
        }
      }
    }
  }
  __syncthreads();
  if (!s_regular) lp_irregular(p, row, t, found.pool, s_sum);
  grid_launch_dependents();
}

}  // namespace fp8gq
