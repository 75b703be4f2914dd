// How many clusters of a launch's shape the machine holds at a time, as the driver has said.  Host code without CUDA.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace adk {

// One kernel's answers.  Any number of threads may ask and keep: an entry is one word, and a lost one is asked for again.
struct ClusterCounts {
  static constexpr uint32_t kEntries = 16;
  unsigned long long entry[kEntries];   // key << 32 | clusters; 0: none
  // device (of 4096), blocks of a cluster (1, 2, 4, 8) and bytes of shared memory (1 to 2^18 - 1), so never 0
  static uint32_t key(int device, uint32_t parts, size_t smem) {
    const uint32_t size = parts == 1 ? 0 : parts == 2 ? 1 : parts == 4 ? 2 : 3;
    return (uint32_t)device << 20 | size << 18 | (uint32_t)smem;
  }
  uint32_t find(uint32_t k) const {   // 0: not known
    for (uint32_t i = 0; i < kEntries; ++i) {
      const unsigned long long e = __atomic_load_n(&entry[i], __ATOMIC_RELAXED);
      if (e >> 32 == k) return (uint32_t)e;
    }
    return 0;
  }
  void keep(uint32_t k, uint32_t clusters) {
    uint32_t at = k * 2654435761u >> 28;   // where all are taken
    for (uint32_t i = 0; i < kEntries; ++i)
      if (__atomic_load_n(&entry[i], __ATOMIC_RELAXED) == 0) {
        at = i;
        break;
      }
    __atomic_store_n(&entry[at], (unsigned long long)k << 32 | clusters, __ATOMIC_RELAXED);
  }
};

}  // namespace adk
