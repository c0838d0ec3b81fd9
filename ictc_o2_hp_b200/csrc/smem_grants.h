// Which kernels have been granted how much dynamic shared memory, and on which device:
// the attribute that raises the limit belongs to the device that is current when it is
// set.  Host only, no CUDA types.
#pragma once

#include <cstddef>
#include <cstdint>

namespace ictc {

class SmemGrants {
 public:
  bool covers(int device, const void* kernel, size_t bytes) const {
    const int at = find(device, kernel);
    return at >= 0 && slots_[at].kernel != nullptr && slots_[at].bytes >= bytes;
  }

  // Remembers a grant; without a slot left for it, the attribute is simply set again on
  // every call.
  void record(int device, const void* kernel, size_t bytes) {
    const int at = find(device, kernel);
    if (at >= 0) slots_[at] = {kernel, device, bytes};
  }

 private:
  static constexpr int kSlots = 4096, kProbes = 64;
  struct Slot {
    const void* kernel;
    int device;
    size_t bytes;
  };

  // The pair's slot, or the free one it would take; -1 when its probes are all taken.
  int find(int device, const void* kernel) const {
    const uint64_t key = reinterpret_cast<uintptr_t>(kernel) + 0x9e3779b97f4a7c15ull * (device + 1);
    const uint32_t start = static_cast<uint32_t>((key * 0xff51afd7ed558ccdull) >> 40);
    for (int i = 0; i < kProbes; ++i) {
      const int at = static_cast<int>((start + i) % kSlots);
      const Slot& s = slots_[at];
      if (s.kernel == nullptr || (s.kernel == kernel && s.device == device)) return at;
    }
    return -1;
  }

  Slot slots_[kSlots] = {};
};

}  // namespace ictc
