// TEST INFRASTRUCTURE ONLY.  Two host threads launch one kernel with different sizes of dynamic LDS at once (gvfi_raise_limit in common.h):
// the limit that is left must be the larger one, whichever thread comes first.
#include "../../gimm-vfi_amd/csrc/common.h"
#include <chrono>
#include <thread>

// The thread that sets its limit first waits (bounded) until the other one has passed its own test of the old limit, or cannot.
// Returns the limit the device ends with; small_first: the smaller request is the first to arrive.
extern "C" int gvfi_emu_limit_selftest(int small_first) {
    std::atomic<int> have{0}, arrived{0}, device{0};
    std::mutex turn;
    auto request = [&](int want, bool late) {
        if (late)
            for (int k = 0; k < 200 && arrived.load() == 0; ++k) std::this_thread::sleep_for(std::chrono::milliseconds(1));
        gvfi_raise_limit(have, turn, want, [&](int n) {
            const int mine = ++arrived;
            // the smaller request's call takes effect last wherever the two can overlap
            if (n == 100) for (int k = 0; k < 200 && (mine == 1 ? arrived.load() < 2 : device.load() != 1000); ++k) std::this_thread::sleep_for(std::chrono::milliseconds(1));
            else for (int k = 0; k < 200 && arrived.load() < 2; ++k) std::this_thread::sleep_for(std::chrono::milliseconds(1));
            if (n == 100) std::this_thread::sleep_for(std::chrono::milliseconds(20));
            device = n;
        });
    };
    std::thread a(request, 100, !small_first), b(request, 1000, (bool)small_first);
    a.join();
    b.join();
    return device.load();
}
