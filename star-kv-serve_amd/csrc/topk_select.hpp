// The k largest of a row of fp32 values and their indices in ascending order, by one workgroup: which
// blocks a query reads, which tokens a cache keeps. Equal values go to the lowest index, NaN counts as
// the largest value and -0 as 0, so the choice is a function of the values alone.
//
// Values are compared as integers of the same order. The k-th largest is found by halving its range
// eight bits at a time: 256 buckets over [least, largest], a histogram in LDS, the bucket that holds it
// becomes the range. Scores of one sign and a few binades spread over the buckets from the first round
// on (buckets of the number's upper bits would put them all in one, whose counter is then added to one
// lane at a time), and two or three rounds do.
#pragma once

#include "common.hpp"

namespace starkv {

__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return v != v ? 0xffffffffu : k;
}

template <int THR>
struct TopkShared {
    uint32_t hist[256];
    uint32_t lo[THR / 64], hi[THR / 64];
    uint32_t bin, above, inside;
    unsigned long long scan[THR / 64];
};

// emit(position, index) for the k values chosen, positions 0 .. k - 1 by ascending index; 0 < k <= count. `key(i)`
// gives value i's key. Every thread of the workgroup calls it.
template <int THR, class Key, class Emit>
__device__ __forceinline__ void topk_ascending(TopkShared<THR>& sh, int count, int k, Key key, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int i = tid; i < count; i += THR) {
        const uint32_t v = key(i);
        lo = min(lo, v);
        hi = max(hi, v);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
    }
    if (lane == 0) {
        sh.lo[wave] = lo;
        sh.hi[wave] = hi;
    }
    __syncthreads();
    for (int w = 0; w < THR / 64; ++w) {
        lo = min(lo, sh.lo[w]);
        hi = max(hi, sh.hi[w]);
    }
    // The values above `hi` are chosen; `need` more come from [lo, hi].
    int need = k;
    bool all = k == count;
    while (!all && lo != hi) {
        const int shift = max(0, 24 - __clz((int)(hi - lo)));
        for (int i = tid; i < 256; i += THR) sh.hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < count; i += THR) {
            const uint32_t v = key(i);
            if (v >= lo && v <= hi) atomicAdd(&sh.hist[(v - lo) >> shift], 1u);
        }
        __syncthreads();
        if (wave == 0) {  // lane: buckets 4 lane .. + 3; from the top, the bucket that passes `need`
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) sum += c[x] = sh.hist[4 * lane + x];
            uint32_t from = sum;  // of this lane's buckets and the lanes above
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = (uint32_t)__shfl_down((int)from, d);
                if (lane + d < 64) from += o;
            }
            uint32_t above = from - sum;
            if (above < (uint32_t)need && from >= (uint32_t)need) {
#pragma unroll
                for (int x = 3; x >= 0; --x) {
                    if (above < (uint32_t)need && above + c[x] >= (uint32_t)need) {
                        sh.bin = 4 * lane + x;
                        sh.above = above;
                        sh.inside = c[x];
                    }
                    above += c[x];
                }
            }
        }
        __syncthreads();
        need -= (int)sh.above;
        lo += sh.bin << shift;
        if (hi - lo >= 1u << shift) hi = lo + ((1u << shift) - 1);
        all = need == (int)sh.inside;  // the bucket whole
    }
    // Chosen: keys above `hi`, and of those in [lo, hi] all, or (one value) the first `need`.
    // A thread takes a run of consecutive indices, so that positions ascend with them.
    const int run = (count + THR - 1) / THR, i0 = min(tid * run, count), i1 = min(i0 + run, count);
    unsigned long long mine = 0;  // chosen above | candidates << 32
    for (int i = i0; i < i1; ++i) {
        const uint32_t v = key(i);
        if (v > hi || (all && v >= lo))
            mine += 1;
        else if (!all && v == lo)
            mine += 1ull << 32;
    }
    unsigned long long incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 63) sh.scan[wave] = incl;
    __syncthreads();
    unsigned long long before = incl - mine;
    for (int w = 0; w < wave; ++w) before += sh.scan[w];
    int sure = (int)(uint32_t)before, ties = (int)(before >> 32);
    for (int i = i0; i < i1; ++i) {
        const uint32_t v = key(i);
        const bool in = v > hi || (all && v >= lo), tie = !in && !all && v == lo;
        if (in || (tie && ties < need)) emit(sure + min(ties, need), i);
        sure += in;
        ties += tie;
    }
}

}  // namespace starkv
