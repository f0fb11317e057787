// What the host side keeps per device.  Nothing of CUDA in here: the tests compile it alone.
#pragma once

#include <atomic>

namespace lc0b200 {

constexpr int kMaxDevices = 64;

// A positive number about a kernel that is asked of the runtime once per device (a static one beside the launch: zeros).
struct PerDeviceNumber {
  std::atomic<int> value[kMaxDevices];
};
// `query()` gives the number, or 0 where it failed: that is not kept, the next call asks again.  Racing first calls both ask.
template <typename Query>
inline int ask_once(PerDeviceNumber& kept, int device, Query query) {
  int value = kept.value[device].load(std::memory_order_acquire);
  if (value == 0) {
    value = query();
    if (value > 0) kept.value[device].store(value, std::memory_order_release);
  }
  return value;
}

}  // namespace lc0b200
