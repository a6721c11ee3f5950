// train_common.hip -- the device of a training call.
#include "train_common.h"

#include <atomic>

namespace vh {

int CallDevice::enter(int ordinal) {
    static std::atomic<uint64_t> seen{0};
    int now = -1;
    if (hipGetDevice(&now) != hipSuccess) {
        (void)hipGetLastError();
        now = -1;
    }
    if (ordinal < 0 || ordinal >= 64 || !((seen.load(std::memory_order_acquire) >> ordinal) & 1)) {
        const int st = open_device(ordinal);  // makes it current
        if (now >= 0 && now != ordinal) {
            if (st == VHIP_OK)
                back = now;
            else
                (void)hipSetDevice(now);
        }
        if (st == VHIP_OK && ordinal < 64) seen.fetch_or(1ull << ordinal, std::memory_order_release);
        return st;
    }
    if (now != ordinal) {
        VH_HIP(hipSetDevice(ordinal));
        back = now;
    }
    return VHIP_OK;
}

}  // namespace vh
