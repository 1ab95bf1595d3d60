// Per-device one-time setup that several host threads may reach at once.
#pragma once

#include <atomic>
#include <mutex>

namespace amass {

// run(dev, set): true when set() has succeeded for device `dev`, here or in an
// earlier call.  One thread runs set(), the others wait for it; a failure is
// returned and the next call tries again.  Devices from 64 on are set up in
// every call.
class DeviceOnce {
 public:
  template <typename F>
  bool run(int dev, F set) {
    const unsigned long long bit =
        dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
    if (done_.load(std::memory_order_acquire) & bit) return true;
    std::lock_guard<std::mutex> hold(mu_);
    if (done_.load(std::memory_order_relaxed) & bit) return true;
    if (!set()) return false;
    done_.fetch_or(bit, std::memory_order_release);
    return true;
  }

 private:
  std::atomic<unsigned long long> done_{0};
  std::mutex mu_;
};

}  // namespace amass
