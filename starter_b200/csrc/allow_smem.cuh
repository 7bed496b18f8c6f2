// The shared memory a kernel may be launched with is an attribute it has on every device by itself: raised where a launch wants more than it was
// raised to there before (asking the driver every time costs a microsecond), and never lowered while another thread's launch may need it.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

template <auto Kernel> static inline int allow_smem(int bytes) {
  static std::atomic<int> allowed[64] = {};
  static std::mutex raising;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  if (device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (allowed[device].load(std::memory_order_acquire) >= bytes) return 0;
  const std::lock_guard<std::mutex> hold(raising);
  if (allowed[device].load(std::memory_order_relaxed) >= bytes) return 0;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) allowed[device].store(bytes, std::memory_order_release);
  return (int)e;
}
