// Work that is done once per device and kept, unless it fails.
#pragma once

#include <atomic>
#include <mutex>

namespace pnv {

constexpr int kMaxDevices = 64;

// once(dev, work): runs `work` (which returns an error code, 0 for none) for the first caller per device, the others wait; what it
// wrote is visible to all after them.  A failure is that call's alone and the next one tries again: a kernel's module may not have
// found the memory to load, which the caller can free.  work must not throw.
class DeviceOnce {
 public:
  template <class Work>
  auto operator()(int dev, Work work) -> decltype(work()) {
    using Code = decltype(work());
    if (done_[dev].load(std::memory_order_acquire)) return Code{};
    const std::lock_guard<std::mutex> lock(mutex_);
    if (done_[dev].load(std::memory_order_relaxed)) return Code{};
    const Code code = work();
    if (code == Code{}) done_[dev].store(true, std::memory_order_release);
    return code;
  }

 private:
  std::mutex mutex_;
  std::atomic<bool> done_[kMaxDevices] = {};
};

}  // namespace pnv
