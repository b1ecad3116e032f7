// Attention of one new token per sequence over a paged key-value cache.
//
// One warp per (sequence, query head): the lanes split the head's values, the
// running maximum and sum of the softmax are kept over one pass.
#pragma once

#include "fp8gq_device.cuh"
#include "rope_append.cuh"

namespace fp8gq {

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_token, q_head;
  CacheView cache;
  const int32_t* table;
  int64_t ld_table;
  int max_pages;
  const int32_t* lens;
  __nv_bfloat16* out;
  int64_t o_token, o_head;
  float* lse;
  int B, Hq, Hkv;
  float scale;
};

template <int N>
__device__ __forceinline__ float dot_warp(const float (&a)[N], const float (&b)[N]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) s += a[e] * b[e];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <int D, bool kFp8>
__global__ void __launch_bounds__(128) paged_decode_kernel(const DecodeParams p) {
  constexpr int N = D / 32;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w < static_cast<int64_t>(p.B) * p.Hq) {
    const int b = static_cast<int>(w / p.Hq), h = static_cast<int>(w % p.Hq);
    const int hk = h / (p.Hq / p.Hkv);
    const int64_t cap = static_cast<int64_t>(p.max_pages) * p.cache.page_size;
    int64_t n = p.lens[b];
    if (n < 0 || n > cap) {
      if (lane == 0) record_error(kSiteBadIndex);
      n = n < 0 ? 0 : cap;
    }
    float q[N], acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      q[e] = __bfloat162float(p.q[b * p.q_token + h * p.q_head + N * lane + e]) * p.scale *
             (kFp8 ? p.cache.k_scale : 1.0f);
      acc[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = 0; j < n; ++j) {
      const int64_t c = j / p.cache.page_size, at = j - c * p.cache.page_size;
      const int64_t page = p.table[b * p.ld_table + c];
      if (page < 0 || page >= p.cache.num_pages) {
        if (lane == 0) record_error(kSiteBadIndex);
        continue;
      }
      const int64_t ko = page * p.cache.k_page + at * p.cache.k_slot + hk * p.cache.k_head + N * lane;
      const int64_t vo = page * p.cache.v_page + at * p.cache.v_slot + hk * p.cache.v_head + N * lane;
      float k[N], v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (kFp8) {
          k[e] = static_cast<float>(static_cast<const __nv_fp8_e4m3*>(p.cache.k)[ko + e]);
          v[e] = static_cast<float>(static_cast<const __nv_fp8_e4m3*>(p.cache.v)[vo + e]) * p.cache.v_scale;
        } else {
          k[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.cache.k)[ko + e]);
          v[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.cache.v)[vo + e]);
        }
      }
      const float s = dot_warp(q, k);
      const float mn = fmaxf(m, s);
      const float a = expf(m - mn), x = expf(s - mn);
      l = l * a + x;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = acc[e] * a + x * v[e];
      m = mn;
    }
    const float r = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e)
      p.out[b * p.o_token + h * p.o_head + N * lane + e] = __float2bfloat16_rn(l > 0.0f ? acc[e] * r : 0.0f);
    if (p.lse && lane == 0) p.lse[w] = l > 0.0f ? m + logf(l) : -INFINITY;
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
