// The dynamic LDS of kernels that take more than a launch may have by itself: each function's limit is raised before its first
// launch, by whichever of several threads comes first.
#pragma once

#include <algorithm>
#include <atomic>
#include <mutex>

#include "common.hpp"

namespace starkv {

class LdsLimits {
public:
    // Allows `fn` that many bytes; STARKV_OK or the error's code.
    int allow(const void* fn, int bytes) {
        if (allowed(fn, count_.load(std::memory_order_acquire)) >= bytes) return STARKV_OK;
        const std::lock_guard<std::mutex> guard(lock_);
        const int n = count_.load(std::memory_order_relaxed);
        if (allowed(fn, n) >= bytes) return STARKV_OK;
        SKV_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (n < MOST) {  // an entry does not change any more once it is counted
            known_[n].fn = fn;
            known_[n].bytes = bytes;
            count_.store(n + 1, std::memory_order_release);
        }
        return STARKV_OK;
    }

private:
    static constexpr int MOST = 256;
    struct Entry { const void* fn; int bytes; };

    int allowed(const void* fn, int n) const {
        int most = -1;
        for (int i = 0; i < n; ++i)
            if (known_[i].fn == fn) most = std::max(most, known_[i].bytes);
        return most;
    }

    Entry known_[MOST] = {};
    std::atomic<int> count_{0};
    std::mutex lock_;
};

}  // namespace starkv
