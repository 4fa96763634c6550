// Which cached tokens a request's newest token sees through a window, by pages of 16 tokens: the decodes over
// 16-bit (window_decode.hip) and 8-bit caches (cache8_decode.hip) share it.
//
// Of a request's L tokens the last one (place L - 1) sees the last `window` and the first `sinks`: place s where
// s >= lo = L - window or s < sinks. The pages that hold such places are taken in order, the first tokens' and
// then the window's, each once; a page is read whole and the places it must not show are masked. No window
// (window = 0) shows all.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

namespace starkv {

struct SeenPages {
    int L, lo, head;    // places [0, head) and [lo, L) are seen, head <= lo
    int first, second;  // pages [0, first) and from `second` on
    int pages;          // both

    __device__ __forceinline__ int page(int i) const { return i < first ? i : i - first + second; }

    // The page's places below x, as a bit each.
    static __device__ __forceinline__ uint32_t below(int x, int pg) { return (1u << min(max(x - 16 * pg, 0), 16)) - 1u; }

    // The places of page pg that are seen.
    __device__ __forceinline__ uint32_t mask(int pg) const { return below(L, pg) & (below(head, pg) | ~below(lo, pg)); }
};

__device__ __forceinline__ SeenPages seen_pages(int L, int window, int sinks) {
    SeenPages s;
    s.L = L;
    s.lo = window > 0 ? max(L - window, 0) : 0;
    s.head = min(sinks, s.lo);
    s.first = (s.head + 15) >> 4;
    s.second = max(s.lo >> 4, s.first);  // a page may hold places of both
    s.pages = s.first + ((L + 15) >> 4) - s.second;
    return s;
}

// The most pages that seen_pages() gives for up to `span` tokens.
inline int seen_pages_most(int span, int window, int sinks) {
    const int all = (int)(((int64_t)span + 15) / 16);
    if (window <= 0) return all;
    return (int)std::min<int64_t>(all, ((int64_t)std::min(sinks, span) + 15) / 16 + ((int64_t)window + 14) / 16 + 1);
}

// The current device's compute units (256 where it does not say).
inline int device_cus() {
    static std::atomic<int> known[64];  // by device: the count does not change, and asking costs a call 0.3 us
    int dev = 0, c = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    c = known[dev].load(std::memory_order_relaxed);
    if (c == 0) {
        if (hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || c <= 0) c = 256;
        known[dev].store(c, std::memory_order_relaxed);
    }
    return c;
}

}  // namespace starkv
