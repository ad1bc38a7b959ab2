// What has to be done once on every device of the process, such as reserving a kernel's shared memory: the limit belongs to the function
// on a device.  Host code without CUDA in it.
#pragma once
#include <atomic>

struct QilPerDevice {
    std::atomic<bool> done[64] = {};
    // Calls `set`, which returns 0 where all is well, unless it has returned 0 on this device before.  Two threads may both call it.
    template <typename Set> auto once(int device, Set set) -> decltype(set()) {
        const bool known = device >= 0 && device < 64;
        if (known && done[device].load(std::memory_order_acquire)) return decltype(set())(0);
        const auto failed = set();
        if (known && !failed) done[device].store(true, std::memory_order_release);
        return failed;
    }
};
