// Host settings that belong to a device (a kernel's attributes) and are made before its first use there.
#pragma once

#include <atomic>
#include <cstdint>

namespace qw {

// Runs `set` unless it has run for this device. Two threads that come first at the same time both do: the settings are the
// same. An exception leaves the device unset.
template <typename F>
void once_per_device(std::atomic<uint64_t>& done, int device, F&& set) {
  const uint64_t bit = device >= 0 && device < 64 ? uint64_t{1} << device : 0;  // others: every time
  if (done.load(std::memory_order_acquire) & bit) return;
  set();
  done.fetch_or(bit, std::memory_order_release);
}

}  // namespace qw
