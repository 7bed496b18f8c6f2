// The shared memory a kernel may be launched with is an attribute it has on every device by itself: set where a launch wants more than was set
// there before (asking the driver every time costs a microsecond).
#pragma once

#include <cuda_runtime.h>

template <auto Kernel> static inline int allow_smem(int bytes) {
  static int allowed[64] = {};               // (two threads at once set the same, or the larger one again)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  if (device >= 0 && device < 64 && allowed[device] >= bytes) return 0;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device >= 0 && device < 64) allowed[device] = bytes;
  return (int)e;
}
