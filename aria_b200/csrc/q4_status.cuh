// q4_status.cuh -- what the entry points of every unit share.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace aria_q4 {

// ARIA_Q4_OK, or ARIA_Q4_ECUDA with the code kept for aria_q4_last_cuda_error
int cuda_status(cudaError_t e);
// ARIA_Q4_OK when the current device is one the library is built for
int check_device();

// multiprocessors of the current device (148 without one)
int sm_count();
// lets Kern use up to `bytes` of dynamic shared memory; asks the driver once per
// kernel and device, so `bytes` is the same at every call
template <auto Kern>
cudaError_t allow_smem(int bytes) {
  constexpr int kMaxDevices = 64;
  static bool done[kMaxDevices] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev >= 0 && dev < kMaxDevices && done[dev]) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  if (dev >= 0 && dev < kMaxDevices) done[dev] = true;
  return cudaSuccess;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace aria_q4
