// What the host finds out or sets once for each device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

namespace nnz {

// An int that belongs to the current device, found on its first use there (not
// 0; two threads that both find it find the same).
class PerDevice {
 public:
  template <typename F>
  int get(F&& find) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMost) return find();
    int n = value_[dev].load(std::memory_order_relaxed);
    if (n == 0) {
      n = find();
      value_[dev].store(n, std::memory_order_relaxed);
    }
    return n;
  }

 private:
  static constexpr int kMost = 64;
  std::atomic<int> value_[kMost] = {};
};

// Raises a kernel's dynamic shared-memory limit, once per device.
inline cudaError_t raise_smem(const void* fn, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace nnz
