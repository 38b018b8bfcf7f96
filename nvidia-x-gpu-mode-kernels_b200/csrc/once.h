// Preparations made once per device (kernel attributes, occupancy): host code
// without CUDA, so that it can be tested on its own.
#pragma once
#include <atomic>
#include <mutex>

namespace nvfp4 {

constexpr int kMaxDevices = 64;

// run(device, f): calls `f` (which returns a status, 0 for success) the first
// time for a device, one thread at a time; f is tried again after a failure.
// Whoever gets 0 sees all that the successful f wrote.  A device index out of
// [0, kMaxDevices) calls f each time.
class OncePerDevice {
 public:
  template <class F>
  int run(int device, F f) {
    if (device < 0 || device >= kMaxDevices) return f();
    if (done_[device].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> lock(mu_);
    if (done_[device].load(std::memory_order_relaxed)) return 0;
    const int status = f();
    if (status == 0) done_[device].store(true, std::memory_order_release);
    return status;
  }

 private:
  std::atomic<bool> done_[kMaxDevices] = {};
  std::mutex mu_;
};

}  // namespace nvfp4
