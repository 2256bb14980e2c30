// How a step flags an index out of bounds.
#pragma once
#include "common.h"
#include "kernels.h"

namespace shk {

// In device memory other flags may be set beside this one. The word in host memory takes no other: a plain
// store (atomics across the bus are not everywhere), which the host reads once the run has ended.
__device__ __forceinline__ void flag_host(uint32_t* host) {
  __hip_atomic_store(host, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__device__ __forceinline__ void flag_out_of_bounds(const FlagWord& f) {
  if (f.host != nullptr) flag_host(f.host);
  else atomicOr(f.status, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS);
}

// The same where a step flags its status word first (one address less in a kernel that is short of registers)
// and hands it on in its last launch, by one thread. A step beside it on another stream may do so with this
// one's flag: the exchange loses none.
__device__ __forceinline__ void hand_on(const FlagWord& f) {
  if (f.host != nullptr && atomicExch(f.status, 0u) != 0u) flag_host(f.host);
}

}  // namespace shk
