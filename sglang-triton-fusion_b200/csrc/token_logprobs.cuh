// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits.  One CTA per row: a pass for the maximum, one for the sums, and one
// per alternative.
#pragma once

#include "fp8gq_device.cuh"

namespace fp8gq {

constexpr int kMaxTop = 32;

struct LogprobParams {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int T, V, K;
};

// A logit and its index as one key: larger logits first, equal ones (0 and -0
// too) by ascending index; NaN above +inf.  0 is below every key.
__device__ __forceinline__ unsigned long long logit_key(float x, int i) {
  uint32_t b = x != x ? 0x7fffffffu : __float_as_uint(x + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
  uint32_t b = static_cast<uint32_t>(key >> 32);
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(row[i]);
  else return row[i];
}

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const LogprobParams p) {
  __shared__ float red[16];
  __shared__ unsigned long long keys[8];
  grid_dependency_wait();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < p.V; i += 256) {
    const float x = logit_at(row, i);
    nan |= x != x;
    m = fmaxf(m, x);
  }
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  nan = __syncthreads_or(nan) != 0;
  m = red[0];
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  __syncthreads();
  const bool bad = nan || isinf(m);
  float s = 0.0f, e = 0.0f;
  for (int i = tid; i < p.V; i += 256) {
    const float y = logit_at(row, i) - m, x = expf(y);
    s += x;
    if (x > 0.0f) e += x * y;
  }
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
  }
  if (lane == 0) {
    red[warp] = s;
    red[8 + warp] = e;
  }
  __syncthreads();
  s = 0.0f;
  e = 0.0f;
  for (int i = 0; i < 8; ++i) {
    s += red[i];
    e += red[8 + i];
  }
  const float lse = bad ? NAN : m + logf(s);
  if (tid == 0) {
    if (p.logprobs) {
      const int64_t tok = p.tokens[t];
      if (tok >= p.V) record_error(kSiteBadIndex);
      p.logprobs[t] = tok < 0 ? 0.0f : tok >= p.V ? NAN : logit_at(row, static_cast<int>(tok)) - lse;
    }
    if (p.entropy) p.entropy[t] = bad ? NAN : logf(s) - e / s;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.K; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.V; i += 256) {
      const unsigned long long key = logit_key(logit_at(row, i), i);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
      best = x > best ? x : best;
    }
    __syncthreads();
    if (lane == 0) keys[warp] = best;
    __syncthreads();
    best = keys[0];
    for (int i = 1; i < 8; ++i) best = keys[i] > best ? keys[i] : best;
    last = best;
    if (tid == 0) {
      p.top_ids[static_cast<int64_t>(t) * p.K + k] = key_index(best);
      p.top_logprobs[static_cast<int64_t>(t) * p.K + k] = key_logit(best) - lse;
    }
  }
  grid_launch_dependents();
}

}  // namespace fp8gq
