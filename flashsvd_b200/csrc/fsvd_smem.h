// A kernel's limit of dynamic shared memory, raised once per device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

namespace fsvd_tile {

// A kernel's dynamic shared-memory limit belongs to a device: raised on the current one, once.
class SmemLimit {
  std::atomic<unsigned long long> raised{0};   // a bit per device
 public:
  template <typename K>
  cudaError_t raise(K* kern, int bytes) {
    return raise_to(kern, [=](int, int& most) {
      most = bytes;
      return cudaSuccess;
    });
  }
  // To all that the device has beside the kernel's own static memory: launches of any size, from any thread, then need
  // nothing more.
  template <typename K>
  cudaError_t raise(K* kern) {
    return raise_to(kern, [=](int dev, int& most) {
      cudaFuncAttributes a;
      cudaError_t e = cudaFuncGetAttributes(&a, reinterpret_cast<const void*>(kern));
      if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
      most -= (int)a.sharedSizeBytes;
      return e;
    });
  }

 private:
  template <typename K, typename F>
  cudaError_t raise_to(K* kern, F limit) {
    int dev = 0, most = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (raised.load(std::memory_order_relaxed) >> dev & 1))) return e;
    e = limit(dev, most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess && dev < 64) raised.fetch_or(1ull << dev);
    return e;
  }
};

}  // namespace fsvd_tile
