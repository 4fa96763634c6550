// The k largest of a row of fp32 values and their indices in ascending order, by one workgroup: which
// blocks a query reads, which tokens a cache keeps. Equal values go to the lowest index, NaN counts as
// the largest value and -0 as 0, so the choice is a function of the values alone.
//
// Values are compared as integers of the same order. 2048 buckets over [least, largest] (scores of one
// sign and a few binades spread over them, where buckets of the number's upper bits would be a handful)
// are counted in LDS; the bucket that holds the k-th largest becomes the range, until it is taken
// whole, holds 64 values or fewer, which one wave ranks, or one value. One round does for most rows.
// A wave takes a run of consecutive values, 64 at a time, so that loads are whole lines and a value's
// place among the chosen is a count of bits; its lanes keep their values in registers (rows past 32768
// values are read again in every pass). The one CU's instructions, barriers and first reads are a row's
// time: 4096 scores 5.3 us from launch to end, where a kernel of three dependent reads and nothing else
// takes 4 (9.0 with a thread's run of consecutive values read from LDS in every pass; 8192 weights 11.2,
// from 17.6).
#pragma once

#include "common.hpp"

namespace starkv {

__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return v != v ? 0xffffffffu : k;
}

// Over the lanes of a wave with data-parallel moves (a cross-lane load through LDS costs a hundred cycles a
// step): the inclusive sum, the least and the largest.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31), c = __builtin_amdgcn_readlane(v, 47);
    const int row = (threadIdx.x >> 4) & 3;
    return v + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

template <int CTL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTL, 0xF, 0xF, true);
}

__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    v = min(v, dpp_u<0xB1>(v));  // as row16_max
    v = min(v, dpp_u<0x4E>(v));
    v = min(v, dpp_u<0x141>(v));
    v = min(v, dpp_u<0x140>(v));
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16),
                   c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return min(min(a, b), min(c, d));
}

// The set lanes of a mask below this one.
__device__ __forceinline__ int lanes_below(unsigned long long mask) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

constexpr int TK_BITS = 11, TK_BINS = 1 << TK_BITS;

constexpr int TK_THR = 1024, TK_WAVES = TK_THR / 64;
// Values a thread keeps, by the longest row: straight code over 4, 16 or 32 of them (a row of 2000 values steps
// over what it does not have of 16 in every pass), longer rows none.
constexpr int TK_FEW = 4, TK_MANY = 16, TK_MOST = 32;

inline int topk_run(int longest) {
    return longest <= TK_THR * TK_FEW ? TK_FEW : longest <= TK_THR * TK_MANY ? TK_MANY : longest <= TK_THR * TK_MOST ? TK_MOST : 0;
}

struct TopkShared {
    uint32_t hist[TK_BINS];
    uint32_t lo[TK_WAVES], hi[TK_WAVES];
    uint32_t above[TK_WAVES];           // values in a wave's buckets
    uint32_t bin, over, inside;
    uint32_t few, key[64], at[64];      // a small bucket's values
    uint32_t sure[TK_WAVES], tie[TK_WAVES];
};

// The sum of t[w] over the waves w after (before) `wave`.
__device__ __forceinline__ uint32_t sum_of_waves(const uint32_t* t, int wave, bool after) {
    static_assert(TK_WAVES == 16, "a wave a lane of a row");
    const int w = threadIdx.x & 15;
    uint32_t v = (after ? w > wave : w < wave) ? t[w] : 0;
    v += dpp_u<0xB1>(v);
    v += dpp_u<0x4E>(v);
    v += dpp_u<0x141>(v);
    return v + dpp_u<0x140>(v);
}

// emit(position, index, value) for the k values chosen of value(0) .. value(count - 1), positions 0 .. k - 1 by
// ascending index; 0 < k <= count, and count <= TK_THR RUN where RUN is not 0. Every thread of the workgroup
// calls it.
template <int RUN, class Value, class Emit>
__device__ __forceinline__ void topk_ascending(TopkShared& sh, int count, int k, Value value, Emit emit) {
    constexpr int PER = TK_BINS / TK_THR;  // buckets a thread
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int run = (count + TK_THR - 1) / TK_THR, i0 = wave * run * 64 + lane;  // the lane's values: i0 + 64 u, u < run
    float kept[RUN ? RUN : 1];
    uint32_t keys[RUN ? RUN : 1];
    if constexpr (RUN) {
#pragma unroll
        for (int u0 = 0; u0 < RUN; u0 += 4)
            if (u0 < run) {
#pragma unroll
                for (int u = u0; u < u0 + 4; ++u) kept[u] = value(min(i0 + 64 * u, count - 1));
            }
    }
    // f(key, index, value) of the lane's values, in order; every lane calls it. A value that the lane has not has
    // key 0, below every value's.
    const auto each = [&](auto f) {
        if constexpr (RUN) {
#pragma unroll
            for (int u0 = 0; u0 < RUN; u0 += 4)
                if (u0 < run) {
#pragma unroll
                    for (int u = u0; u < u0 + 4; ++u) f(keys[u], i0 + 64 * u, kept[u]);
                }
        } else {
            constexpr int AT_ONCE = 16;  // reads on their way
            for (int u0 = 0; u0 < run; u0 += AT_ONCE) {
                float v[AT_ONCE];
#pragma unroll
                for (int x = 0; x < AT_ONCE; ++x) v[x] = value(min(i0 + 64 * (u0 + x), count - 1));
#pragma unroll
                for (int x = 0; x < AT_ONCE; ++x) {
                    const int i = i0 + 64 * (u0 + x);
                    f(u0 + x < run && i < count ? order_key(v[x]) : 0, i, v[x]);
                }
            }
        }
    };
#pragma unroll
    for (int x = 0; x < PER; ++x) sh.hist[x * TK_THR + tid] = 0;
    if (tid == 0) sh.few = 0;
    uint32_t lo = 0xffffffffu, hi = 0;
    if constexpr (RUN) {
#pragma unroll
        for (int u0 = 0; u0 < RUN; u0 += 4)
            if (u0 < run) {
#pragma unroll
                for (int u = u0; u < u0 + 4; ++u) {
                    const uint32_t v = order_key(kept[u]);  // of a lane's own or the row's last value
                    lo = min(lo, v);
                    hi = max(hi, v);
                    keys[u] = u < run && i0 + 64 * u < count ? v : 0;
                }
            }
    } else {
        each([&](uint32_t v, int, float) {
            lo = min(lo, v ? v : lo);
            hi = max(hi, v);
        });
    }
    lo = wave_least(lo);
    hi = ~wave_least(~hi);
    if (lane == 0) {
        sh.lo[wave] = lo;
        sh.hi[wave] = hi;
    }
    __syncthreads();
    lo = wave_least(sh.lo[lane & 15]);
    hi = ~wave_least(~sh.hi[lane & 15]);
    // The values above `hi` are chosen; `need` more come from [lo, hi]: all of them, the first `need` of one
    // value's, or those before (key, index) = (lo, limit).
    int need = k, limit = -1;
    bool all = k == count;
    while (!all && lo != hi) {
        const int shift = max(0, 32 - TK_BITS - __clz((int)(hi - lo)));
        each([&](uint32_t v, int, float) {
            if (v - lo <= hi - lo) atomicAdd(&sh.hist[(v - lo) >> shift], 1u);
        });
        __syncthreads();
        // From the top, the bucket that passes `need`: a thread's buckets, its wave's, the waves above.
        uint32_t c[PER], sum = 0;
#pragma unroll
        for (int x = 0; x < PER; ++x) sum += c[x] = sh.hist[tid * PER + x];
        const uint32_t upto = wave_prefix(sum), whole = __builtin_amdgcn_readlane(upto, 63);
        if (lane == 0) sh.above[wave] = whole;
        __syncthreads();
        uint32_t over = whole - upto + sum_of_waves(sh.above, wave, true);
        if (over < (uint32_t)need && over + sum >= (uint32_t)need) {
#pragma unroll
            for (int x = PER - 1; x >= 0; --x) {
                if (over < (uint32_t)need && over + c[x] >= (uint32_t)need) {
                    sh.bin = tid * PER + x;
                    sh.over = over;
                    sh.inside = c[x];
                }
                over += c[x];
            }
        }
#pragma unroll
        for (int x = 0; x < PER; ++x) sh.hist[tid * PER + x] = 0;
        __syncthreads();
        need -= (int)sh.over;
        lo += sh.bin << shift;
        if (hi - lo >= 1u << shift) hi = lo + ((1u << shift) - 1);
        const int inside = (int)sh.inside;
        all = need == inside;  // the bucket whole
        if (all || inside > 64) continue;
        each([&](uint32_t v, int i, float) {
            if (v - lo <= hi - lo) {
                const uint32_t s = atomicAdd(&sh.few, 1u);
                sh.key[s] = v;
                sh.at[s] = i;
            }
        });
        __syncthreads();
        if (wave == 0) {  // a lane's value has as many before it as are larger, or equal at a lower index
            const uint32_t v = lane < inside ? sh.key[lane] : 0, at = lane < inside ? sh.at[lane] : 0;
            int before = 0;
            for (int i = 0; i < inside; ++i) {
                const uint32_t o = __builtin_amdgcn_readlane(v, i), oat = __builtin_amdgcn_readlane(at, i);
                before += o > v || (o == v && oat < at);
            }
            if (lane < inside && before == need - 1) {  // the last one chosen
                sh.bin = v;
                sh.over = at;
            }
        }
        __syncthreads();
        lo = hi = sh.bin;
        limit = (int)sh.over;
    }
    const bool first = !all && limit < 0;  // the first `need` of the values equal to lo
    if (all) hi = lo - 1;                  // all from lo on; one that equals hi comes after `limit`
    const auto sure = [&](uint32_t v, int i) { return v > hi || (v == hi && i <= limit); };
    int chosen = 0, ties = 0;  // of the wave's values
    each([&](uint32_t v, int i, float) {
        chosen += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sure(v, i)));
        if (first) ties += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v == hi));
    });
    if (lane == 0) {
        sh.sure[wave] = chosen;
        sh.tie[wave] = ties;
    }
    __syncthreads();
    chosen = (int)sum_of_waves(sh.sure, wave, false);
    ties = (int)sum_of_waves(sh.tie, wave, false);
    each([&](uint32_t v, int i, float x) {
        const bool s = sure(v, i);
        const unsigned long long in = __builtin_amdgcn_ballot_w64(s);
        if (!first) {
            if (s) emit(chosen + lanes_below(in), i, x);
        } else {
            const unsigned long long equal = __builtin_amdgcn_ballot_w64(v == hi);
            const int before = ties + lanes_below(equal);
            if (s || (v == hi && before < need)) emit(chosen + lanes_below(in) + min(before, need), i, x);
            ties += __builtin_popcountll(equal);
        }
        chosen += __builtin_popcountll(in);
    });
}

}  // namespace starkv
