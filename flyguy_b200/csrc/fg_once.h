// What has to be set up once on every device of a process. Host code.
#pragma once
#include <stdint.h>

#include <atomic>

namespace fgm {

// A kernel's opt-in to more shared memory belongs to a device, and may be asked for by two threads at once: f runs at a device's
// first call, and again only if it threw (or two threads came first). Devices from 64 on: at every call.
class OnEachDevice {
  public:
    template <class F>
    void first(int device, F&& f) {
        const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
        if (done_.load(std::memory_order_acquire) & bit) return;
        f();
        done_.fetch_or(bit, std::memory_order_release);
    }

  private:
    std::atomic<uint64_t> done_{0};
};

}  // namespace fgm
