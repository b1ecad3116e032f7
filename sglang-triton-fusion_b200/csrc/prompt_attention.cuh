// Attention over packed prompts.
//
// One warp per (query row, head): the lanes split the head's values, the
// running maximum and sum of the softmax are kept over one pass.
#pragma once

#include "fp8gq_device.cuh"
#include "paged_decode.cuh"

namespace fp8gq {

struct PromptParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, Tq, Tk, Hq, Hkv;
  float scale;
  int causal;
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

__device__ __forceinline__ int cut(int x, int hi) {
  if (x < 0 || x > hi) {
    record_error(kSiteBadIndex);
    return x < 0 ? 0 : hi;
  }
  return x;
}

template <int D>
__global__ void __launch_bounds__(128) prompt_attention_kernel(const PromptParams p) {
  constexpr int N = D / 32;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int row = static_cast<int>(w / p.Hq), h = static_cast<int>(w % p.Hq);
  if (row < p.Tq) {
    int b = 0;
    while (b < p.B && !(row >= cut(p.cu_q[b], p.Tq) && row < cut(p.cu_q[b + 1], p.Tq))) ++b;
    if (b < p.B) {
      const int hk = h / (p.Hq / p.Hkv);
      const int q0 = cut(p.cu_q[b], p.Tq), q1 = cut(p.cu_q[b + 1], p.Tq);
      const int k0 = cut(p.cu_k[b], p.Tk), k1 = cut(p.cu_k[b + 1], p.Tk);
      if (k1 < k0) record_error(kSiteBadIndex);
      int n = k1 - k0;
      if (p.causal) n = min(n, row - q0 + (k1 - k0) - (q1 - q0) + 1);
      float q[N], acc[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        q[e] = __bfloat162float(p.q[row * p.q_token + h * p.q_head + N * lane + e]) * p.scale;
        acc[e] = 0.0f;
      }
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < n; ++j) {
        float k[N], v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          k[e] = __bfloat162float(p.k[(k0 + j) * p.k_token + hk * p.k_head + N * lane + e]);
          v[e] = __bfloat162float(p.v[(k0 + j) * p.v_token + hk * p.v_head + N * lane + e]);
        }
        const float s = dot_warp(q, k);
        const float mn = fmaxf(m, s);
        const float a = expf(m - mn), x = expf(s - mn);
        l = l * a + x;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = acc[e] * a + x * v[e];
        m = mn;
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
        p.out[row * p.o_token + h * p.o_head + N * lane + e] = __float2bfloat16_rn(l > 0.0f ? acc[e] / l : 0.0f);
      if (p.lse && lane == 0) p.lse[w] = l > 0.0f ? m + logf(l) : -INFINITY;
    }
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
