// dgs_guard.cuh -- a kernel's report of an id it met outside its source (device only).
#pragma once

#include "dgs_common.h"

namespace dgs {

// Stores the first out-of-range id a launch met into the process's async error words
// (context.h): id, row count and call tag first, then the kind with a system-scope release.
static __device__ __attribute__((noinline)) void report_bad_id(int64_t *err, int64_t kind,
                                                               int64_t id, uint64_t rows,
                                                               int64_t tag) {
  __hip_atomic_store(err + 1, id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  __hip_atomic_store(err + 2, (int64_t)rows, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  __hip_atomic_store(err + 3, tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  __hip_atomic_store(err, kind, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

}  // namespace dgs
