// What the translation units with extern "C" entry points share: error texts, the launch counter and
// small host-side checks.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "megaslide_b200.h"

namespace msl {

// Records a formatted description for msl_last_error() and returns `code`.
int failf(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Adds to msl_launch_count().
void count_launches(unsigned n);

inline int cuda_failf(cudaError_t e, const char* what) {
  return failf(MSL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline bool multiple_of(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// SMs of the current device (cached per device; 148 on a B200).
int sm_count();

}  // namespace msl
