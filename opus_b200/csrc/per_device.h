// Answers of the driver that are asked for once for each device (no CUDA here: it compiles with any C++ compiler).
#pragma once

#include <atomic>

namespace opus {

// Positive numbers by device and key in [0, Keys).  A query that fails (below 1) is not kept: it is asked again.
template <int Keys>
class PerDevice {
 public:
  template <typename Query>
  int get(int device, int key, int fallback, Query query) {
    const bool kept = device >= 0 && device < kDevices;
    int n = kept ? known_[device][key].load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    n = query();
    if (n < 1) return fallback;
    if (kept) known_[device][key].store(n, std::memory_order_relaxed);
    return n;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices][Keys] = {};
};

}  // namespace opus
