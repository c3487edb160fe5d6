// Error flags that several devices hold, read from the host.
#pragma once

#include <stdint.h>

#include <atomic>

namespace shahd {

// Devices 0 .. 63 that something has been launched on.
struct DeviceSet {
  std::atomic<uint64_t> bits{0};
  void Add(int device) { bits.fetch_or(uint64_t(1) << device, std::memory_order_relaxed); }
};

// The first flag that is not 0, in the order of the devices; -1 for one that read(device, &flag) cannot read.
template <class Read>
int FirstFlag(const DeviceSet& devices, Read&& read) {
  const uint64_t bits = devices.bits.load(std::memory_order_relaxed);
  for (int device = 0; device < 64; device++) {
    if (!(bits >> device & 1)) continue;
    int flag = 0;
    if (!read(device, &flag)) flag = -1;
    if (flag != 0) return flag;
  }
  return 0;
}

}  // namespace shahd
