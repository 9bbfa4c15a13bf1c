// What a launch asks of its device, looked up once.
#pragma once

#include <atomic>

#include <cuda_runtime.h>

namespace dsalt {

// SMs of the current device.  Launches come from any thread at any time: threads that
// both find no entry both write the same one.
inline cudaError_t sm_count(int* out) {
  static std::atomic<int> counts[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int n = counts[dev].load(std::memory_order_relaxed);
  if (n <= 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    counts[dev].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return cudaSuccess;
}

}  // namespace dsalt
