// Host helpers shared by the library's translation units: device checks, the
// status of a failed CUDA call, the tensor-map encoder and the shared-memory
// opt-in.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>

#include "../../include/fp8gq.h"

namespace fp8gq {

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  int sm_count = 0;
  int cc_major = 0;
  int max_smem_optin = 0;
};

inline int device_info(DeviceInfo* out, int* dev_out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return FP8GQ_ERR_DEVICE;
  static std::mutex mu;
  static DeviceInfo info[kMaxDevices];
  std::lock_guard<std::mutex> lk(mu);
  DeviceInfo& d = info[dev];
  if (d.sm_count == 0) {
    if (cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&d.max_smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) !=
            cudaSuccess) {
      d.sm_count = 0;
      return FP8GQ_ERR_DEVICE;
    }
  }
  if (d.cc_major != 10) return FP8GQ_ERR_DEVICE;
  *out = d;
  if (dev_out) *dev_out = dev;
  return FP8GQ_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// FP8GQ_ERR_LAUNCH for a failed CUDA call; with FP8GQ_DEBUG set in the
// environment the CUDA error is also printed to stderr.
inline int cuda_fail(cudaError_t e, const char* what) {
  static const bool debug = std::getenv("FP8GQ_DEBUG") != nullptr;
  if (debug) std::fprintf(stderr, "fp8gq: %s: %s\n", what, cudaGetErrorString(e));
  return FP8GQ_ERR_LAUNCH;
}

inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? FP8GQ_OK : FP8GQ_ERR_LAUNCH;
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// cudaFuncAttributeMaxDynamicSharedMemorySize raised to the device's limit
// once per kernel and device (launches then pass their own smaller sizes).
inline cudaError_t ensure_max_smem(const void* fn, int max_smem) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const auto key = std::make_pair(dev, fn);
  {
    std::lock_guard<std::mutex> lock(mu);
    auto it = done.find(key);
    if (it != done.end() && it->second >= max_smem) return cudaSuccess;
  }
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  done[key] = max_smem;
  return cudaSuccess;
}

// cudaFuncAttributeNonPortableClusterSizeAllowed set once per kernel and
// device, before a cluster of more than 8 CTAs is queried or launched.
inline cudaError_t ensure_nonportable_clusters(const void* fn) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, bool> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const auto key = std::make_pair(dev, fn);
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(key)) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done[key] = true;
  return e;
}

// The error word and the wait limit are device variables, of which each
// translation unit with bounded waits has its own; these read, clear and set
// the serving operators' (serve_api.cu), for fp8gq_device_error and
// fp8gq_set_wait_limit_ns.
int serve_error_word(unsigned int* code, int clear);
int serve_set_wait_limit(unsigned long long limit_ns);

}  // namespace fp8gq
