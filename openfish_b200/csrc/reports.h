// reports.h -- who has been told that kernels on a device have given up waiting: plain C++, so that it can be tried without a GPU.
//
// The kernels count on the device how often they have given up; nothing there is ever cleared, so nothing that happens beside a look is lost.  Every
// host thread remembers the count it was last told, so that one thread's look takes no other's report away.
#pragma once
#include <atomic>

struct Reports {
    static constexpr int kDevices = 64;
    std::atomic<int> latest[kDevices] = {};  // the count that any thread has read last

    // `known`: the calling thread's memory, kDevices numbers, zeros at first (else the count it was told, and one).
    // A thread's first call of an operator: what has been reported by then is no concern of its kernels.
    void begin(int device, int *known) {
        if (device < kDevices && !known[device]) known[device] = latest[device].load(std::memory_order_relaxed) + 1;
    }
    // The thread has read `count`: whether that is news to it.  (A count of zero: nothing yet, or the device was reset.)
    bool take(int device, int *known, int count) {
        if (device >= kDevices) return count != 0;
        begin(device, known);
        const bool news = count != 0 && count + 1 != known[device];
        known[device] = count + 1;
        latest[device].store(count, std::memory_order_relaxed);
        return news;
    }
};
