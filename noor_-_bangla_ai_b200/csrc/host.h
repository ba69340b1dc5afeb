// host.h -- what the library's host code shares: the last-error message, the
// status macros, the device guard and the shared-memory limit of kernels.
#pragma once

#include <cuda_runtime.h>

#include <mutex>
#include <vector>

#include "noor_moe.h"

namespace noor {

// Records the thread's last-error message (noor_moe_last_error) and returns
// `code`.
int fail(int code, const char* fmt, ...);

// A failed runtime call is reported by the call that made it; the runtime's
// last-error state is cleared so that it does not resurface as the launch
// error of a later, unrelated call (faults that poison the context stay).
#define CK(call)                                                                                       \
  do {                                                                                                 \
    cudaError_t e_ = (call);                                                                           \
    if (e_ != cudaSuccess) {                                                                           \
      (void)cudaGetLastError();                                                                        \
      return noor::fail(e_ == cudaErrorMemoryAllocation ? NOOR_MOE_ERR_OOM : NOOR_MOE_ERR_CUDA,        \
                        "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__);          \
    }                                                                                                  \
  } while (0)

#define CKR(call)               \
  do {                          \
    int rc_ = (call);           \
    if (rc_ != NOOR_MOE_OK) return rc_; \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

// Raise a kernel's dynamic shared-memory limit to at least `bytes`.  Up to
// 48 KB needs no attribute; above it the limit set so far for each
// (kernel, device) is remembered, so the slow host call runs only when a
// launch needs more than before.
template <typename K>
int ensure_smem_limit(K kern, int bytes) {
  if (bytes <= 48 * 1024) return NOOR_MOE_OK;
  static std::mutex mu;
  struct Entry {
    const void* kern;
    int dev;
    int bytes;
  };
  static std::vector<Entry> done;
  int dev = 0;
  CK(cudaGetDevice(&dev));
  const void* key = reinterpret_cast<const void*>(kern);
  std::lock_guard<std::mutex> lock(mu);
  for (auto& e : done)
    if (e.kern == key && e.dev == dev) {
      if (e.bytes >= bytes) return NOOR_MOE_OK;
      CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      e.bytes = bytes;
      return NOOR_MOE_OK;
    }
  CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.push_back({key, dev, bytes});
  return NOOR_MOE_OK;
}

}  // namespace noor
