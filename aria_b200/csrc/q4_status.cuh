// q4_status.cuh -- what the entry points of every unit share.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace aria_q4 {

// ARIA_Q4_OK, or ARIA_Q4_ECUDA with the code kept for aria_q4_last_cuda_error
int cuda_status(cudaError_t e);
// ARIA_Q4_OK when the current device is one the library is built for
int check_device();

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace aria_q4
