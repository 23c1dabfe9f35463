// Host-side launch set-up that the kernels with large shared memory have in common.
#pragma once

#include <cuda_runtime.h>

#include <mutex>

namespace dsv4 {

// Let KERNEL use `bytes` of dynamic shared memory on the current device (a per-device attribute of a
// kernel: set once for each).  `device`, if not null, receives the current device.
template <auto KERNEL>
cudaError_t allow_shared_memory(size_t bytes, int* device = nullptr) {
  constexpr int MAX_DEVICES = 64;
  static std::mutex mu;
  static bool configured[MAX_DEVICES] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e) return e;
  if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
  if (device != nullptr) *device = dev;
  std::lock_guard<std::mutex> lk(mu);
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e) return e;
    configured[dev] = true;
  }
  return cudaSuccess;
}

}  // namespace dsv4
