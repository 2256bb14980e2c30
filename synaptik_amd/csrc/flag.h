// Flags an index out of bounds in the word that a run reports.
#pragma once
#include "common.h"
#include "kernels.h"

namespace shk {

// In device memory other flags may be set beside this one. A word in host memory takes no other: a plain
// store (atomics across the bus are not everywhere), which the host reads once the run has ended.
__device__ __forceinline__ void flag_out_of_bounds(const FlagWord& f) {
  if (f.host) __hip_atomic_store(f.word, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  else atomicOr(f.word, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS);
}

}  // namespace shk
