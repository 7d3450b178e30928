// What has to follow a store wider than 64 bits.
#pragma once

#include <hip/hip_runtime.h>

namespace osm {

// A vector instruction that overwrites the data registers of a store wider than
// 64 bits right after it was seen on MI355X to corrupt the store's first dword now
// and then (the compiler placed no wait state there).  Two wait states, which no
// instruction can be scheduled into or ahead of.
__device__ __forceinline__ void wide_store_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 1" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace osm
