// Checks of the C entry points' arguments.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
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

// SMs of a device, asked for once (148 without one, so that sizes can be computed anywhere)
inline int device_sms(int dev) {
  static std::atomic<int> known[64];
  if (dev >= 0 && dev < 64) {
    const int n = known[dev].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int n = 0;
  if (dev < 0 || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace yb
