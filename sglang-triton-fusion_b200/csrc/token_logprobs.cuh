// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits.
//
// Mathematics: with m the row's maximum, s = sum exp(x - m) and
// e = sum exp(x - m) (x - m):  logprob(t) = (x_t - m) - log s,
// entropy = log s - e / s.  Each thread keeps (m, s, e) of what it has read,
// rescaled when m moves; such triples join in any grouping.  The alternatives
// are kept the same way: each warp holds its best top_k sorted across its
// lanes; sorted lists join pairwise.
//
// Bound: HBM, one pass (5 fp32 operations and one exponential per value).
//
// A row is read by a cluster of 1 to 16 CTAs (more for fewer rows), joined over
// distributed shared memory: one launch, no scratch.  A value reaches the
// sorted list only if it beats a threshold -- the list's last entry, or a lower
// bound of the row's top_k-th value that any warp of the CTA has found -- so
// that after the first chunk, whose threshold is the top_k-th largest of the
// lanes' maxima, few do.  Joins and sums have a fixed order; the threshold only
// spares work, so results do not depend on timing.
#pragma once

#include "fp8gq_device.cuh"
#include "tensor_core.cuh"

namespace fp8gq {

constexpr int kMaxTop = 32;
constexpr int kLpWarps = 8;
constexpr int kLpThreads = 32 * kLpWarps;
constexpr int kLpUnroll = 4;              // 16-byte vectors per lane and chunk
constexpr float kLpFar = -1000.0f;        // exp(x - m) is 0 long before: stands for any smaller difference, -inf too

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

template <typename T>
__device__ __forceinline__ void lp_unpack(float (&x)[16 / sizeof(T)], uint4 a) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

struct LpSums {
  float m, s, e;
};
__device__ __forceinline__ void lp_move(LpSums& a, float m) {
  const float d = fmaxf(a.m - m, kLpFar), f = lp_ex2(d * kLog2e);
  a.e = (a.e + d * a.s) * f;
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void lp_add(LpSums& a, float x) {
  const float y = max_nan(x - a.m, kLpFar), f = lp_ex2(y * kLog2e);
  a.s += f;
  a.e = __fmaf_rn(f, y, a.e);
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

// A warp's best values, entry i on lane i.
struct LpList {
  float v;       // this lane's entry
  int id;
  float kv;      // the last (top_k-th) entry, on every lane
  int kid;
};

// Offers x (index id) of every lane: those above thr enter.  Equal values order
// by index, so entries may come in any order.
__device__ __forceinline__ void lp_offer(LpList& l, float x, int id, float& thr, int K, int lane) {
  bool c = x > thr || (x == l.kv && id < l.kid && x > -INFINITY);
  unsigned b = __ballot_sync(0xffffffffu, c);
  while (b) {
    const int src = __ffs(b) - 1;
    const float cx = __shfl_sync(0xffffffffu, x, src);
    const int cid = __shfl_sync(0xffffffffu, id, src);
    const int pos = __popc(__ballot_sync(0xffffffffu, l.v > cx || (l.v == cx && l.id < cid)));
    const float uv = __shfl_up_sync(0xffffffffu, l.v, 1);
    const int uid = __shfl_up_sync(0xffffffffu, l.id, 1);
    if (lane > pos) {
      l.v = uv;
      l.id = uid;
    } else if (lane == pos) {
      l.v = cx;
      l.id = cid;
    }
    l.kv = __shfl_sync(0xffffffffu, l.v, K - 1);
    l.kid = __shfl_sync(0xffffffffu, l.id, K - 1);
    thr = fmaxf(thr, l.kv);
    c = c && lane != src && (x > thr || (x == l.kv && id < l.kid && x > -INFINITY));
    b = __ballot_sync(0xffffffffu, c);
  }
}

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

// The K-th largest of the lanes' values (no NaN).
__device__ __forceinline__ float lp_kth_lane(float v, int K, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int x = k >> 1; x > 0; x >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, x);
      const bool keep_max = ((lane & x) == 0) == ((lane & k) == 0);
      v = keep_max ? fmaxf(v, o) : fminf(v, o);
    }
  return __shfl_sync(0xffffffffu, v, K - 1);
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobParams p) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ lp_key s_list[kLpWarps][32];
  __shared__ lp_key s_out[32];
  __shared__ LpSums s_sum[kLpWarps], s_total;
  __shared__ int s_tau;
  __shared__ int s_nan;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int t = blockIdx.x / p.cluster;
  const int K = p.K;
  if (tid == 0) s_tau = kOrderMinusInf;
  __syncthreads();
  grid_dependency_wait();

  // a row: up to kVec - 1 values before the first 16-byte boundary, vectors, up to kVec - 1 after
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  const int before = min(p.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (p.V - before) / kVec;
  const int after0 = before + vectors * kVec;
  const uint4* vec = reinterpret_cast<const uint4*>(row + before);
  const int v_lo = static_cast<int>(static_cast<int64_t>(vectors) * rank / p.cluster);
  const int v_hi = static_cast<int>(static_cast<int64_t>(vectors) * (rank + 1) / p.cluster);

  LpSums sum = {-3.402823466e38f, 0.0f, 0.0f};
  LpList list = {-INFINITY, 0x7fffffff, -INFINITY, 0x7fffffff};
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  bool first = true;
  for (int v0 = v_lo + warp * 32 * kLpUnroll; v0 < v_hi; v0 += kLpThreads * kLpUnroll) {
    uint4 raw[kLpUnroll];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int v = v0 + 32 * u + lane;
      raw[u] = v < v_hi ? __ldcs(vec + v) : make_uint4(none, none, none, none);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float x[kVec];
      lp_unpack<T>(x, raw[u]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) mx = fmaxf(mx, x[i]);
    }
    if (mx > sum.m) lp_move(sum, mx);
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float x[kVec];
      lp_unpack<T>(x, raw[u]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) lp_add(sum, x[i]);
    }
    if (K > 0) {
      float thr = fmaxf(list.kv, just_below(*reinterpret_cast<volatile int*>(&s_tau)));
      if (__any_sync(0xffffffffu, mx > thr)) {
        if (first) thr = fmaxf(thr, just_below(float_order(lp_kth_lane(mx, K, lane))));
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          float x[kVec];
          lp_unpack<T>(x, raw[u]);
          const int id = before + (v0 + 32 * u + lane) * kVec;
#pragma unroll
          for (int i = 0; i < kVec; ++i) lp_offer(list, x[i], id + i, thr, K, lane);
        }
        if (lane == 0) atomicMax(&s_tau, float_order(list.kv));
      }
      first = false;
    }
  }
  // the values outside the vectors: one per lane of one warp
  if (warp == 0 && rank == 0) {
    const int id = lane < 8 ? lane : after0 + lane - 8;
    const bool has = lane < 8 ? lane < before : id < p.V && lane < 16;
    const float x = has ? logit_at(row, id) : -INFINITY;
    if (x > sum.m) lp_move(sum, x);
    lp_add(sum, x);
    if (K > 0) {
      float thr = list.kv;
      lp_offer(list, has ? x : -INFINITY, has ? id : 0x7fffffff, thr, K, lane);
    }
  }

  // ---- the warps, then the cluster's CTAs, in order ----
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    const LpSums o = lp_shfl_xor(sum, x);
    if (lane & x) {                       // the same order of the two on both lanes
      LpSums a = o;
      lp_join(a, sum);
      sum = a;
    } else {
      lp_join(sum, o);
    }
  }
  if (lane == 0) s_sum[warp] = sum;
  lp_key key = list.v > -INFINITY && lane < K ? logit_key(list.v, list.id) : 0;
  s_list[warp][lane] = key;
  if (K > 0) key = lp_merge_lists(s_list, warp, lane);
  else __syncthreads();
  if (warp == 0) {
    if (lane == 0) {
      sum = s_sum[0];
      for (int w = 1; w < kLpWarps; ++w) lp_join(sum, s_sum[w]);
      s_total = sum;
    }
    s_out[lane] = key;
  }
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
        __syncthreads();
        s_list[warp][lane] = a;
        key = lp_merge_lists(s_list, warp, lane);
      }
      if (warp == 0) {
        LpSums o = {-3.402823466e38f, 0.0f, 0.0f};
        if (lane < p.cluster) {
          o.m = ld_dsmem(dsmem_addr(&s_total.m, lane));
          o.s = ld_dsmem(dsmem_addr(&s_total.s, lane));
          o.e = ld_dsmem(dsmem_addr(&s_total.e, lane));
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
          const LpSums q = lp_shfl_xor(o, x);
          if (lane & x) {
            LpSums a = q;
            lp_join(a, o);
            o = a;
          } else {
            lp_join(o, q);
          }
        }
        sum = o;
      }
    }
    cluster_sync_all();                   // the others' shared memory has been read
    if (rank != 0) {
      grid_launch_dependents();
      return;
    }
  }

  // ---- results: warp 0 of the first CTA ----
  if (warp == 0) {
    sum.m = __shfl_sync(0xffffffffu, sum.m, 0);
    sum.s = __shfl_sync(0xffffffffu, sum.s, 0);
    sum.e = __shfl_sync(0xffffffffu, sum.e, 0);
    const bool nan = sum.s != sum.s;      // a NaN or +inf among the values
    const float log_s = nan || sum.s == 0.0f ? NAN : logf(sum.s);
    if (lane == 0) {
      if (p.logprobs) {
        const int64_t tok = p.tokens[t];
        if (tok >= p.V) record_error(kSiteBadIndex);
        p.logprobs[t] = tok < 0 ? 0.0f : tok >= p.V ? NAN : (logit_at(row, tok) - sum.m) - log_s;
      }
      if (p.entropy) p.entropy[t] = log_s - sum.e / sum.s;
      s_nan = nan;
    }
    if (K > 0 && !nan) {
      // fewer than K tokens above -inf: the first of the others follow, which
      // are among the first K
      const int n = __popc(__ballot_sync(0xffffffffu, key != 0 && lane < K));
      if (n < K) {
        bool in = false;
        for (int i = 0; i < n; ++i) in |= key_index(__shfl_sync(0xffffffffu, key, i)) == lane;
        const unsigned free = __ballot_sync(0xffffffffu, !in && lane < K);
        // entry n + r is the r-th free index
        int at = lane >= n ? lane - n : 0, idx = 0;
        unsigned f = free;
        for (int i = 0; i < at; ++i) f &= f - 1;
        idx = __ffs(f) - 1;
        if (lane >= n && lane < K) key = logit_key(-INFINITY, idx);
      }
      if (lane < K) {
        p.top_ids[static_cast<int64_t>(t) * K + lane] = key_index(key);
        p.top_logprobs[static_cast<int64_t>(t) * K + lane] = (key_logit(key) - sum.m) - log_s;
      }
    }
  }
  if (K > 0) {
    __syncthreads();
    if (s_nan) {
      // a row with NaN or +inf: its order alone, one pass per alternative
      lp_key last = ~0ull;
      for (int k = 0; k < K; ++k) {
        lp_key best = 0;
        for (int i = tid; i < p.V; i += kLpThreads) {
          const lp_key x = logit_key(logit_at(row, i), i);
          if (x < last && x > best) best = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const lp_key x = __shfl_xor_sync(0xffffffffu, best, o);
          best = x > best ? x : best;
        }
        __syncthreads();
        if (lane == 0) s_out[warp] = best;
        __syncthreads();
        best = s_out[0];
        for (int i = 1; i < kLpWarps; ++i) best = s_out[i] > best ? s_out[i] : best;
        last = best;
        if (tid == 0) {
          p.top_ids[static_cast<int64_t>(t) * K + k] = key_index(best);
          p.top_logprobs[static_cast<int64_t>(t) * K + k] = NAN;
        }
      }
    }
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
