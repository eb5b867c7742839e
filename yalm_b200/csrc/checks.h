// Checks of the C entry points' arguments.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <string>
#include <utility>

#include "engine.h"

namespace yb {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Every buffer must be memory that the current device `dev` can read: a host pointer or another device's
// memory is refused here instead of faulting in the kernel.
inline int check_device(int dev, std::initializer_list<std::pair<const char*, const void*>> bufs) {
  for (const auto& b : bufs) {
    if (!b.second) continue;
    cudaPointerAttributes at;
    YB_CK(cudaPointerGetAttributes(&at, b.second));
    if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
      return set_error(YB_E_INVALID, std::string(b.first) + " is not memory of the current device");
  }
  return 0;
}

}  // namespace yb
