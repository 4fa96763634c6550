// One token's attention over an 8-bit cache (cache8.hpp has what it holds), whole or through a window
// (window_pages.hpp), on matrix instructions.
//
// For a request b, a KV head h and its G <= 16 query heads, over the places t that the newest token sees, with K_t =
// k_t 2^a, V_t = v_t 2^c (k, v codes; a, c the exponents of t's block):
//     s_t = scale log2(e) 2^a (q . k_t),  out = sum_t 2^(s_t - m) 2^c v_t / sum_t 2^(s_t - m).
// Codes are never multiplied by their scales: 2^a goes onto the 4 scores that a lane has of a page, 2^c into its
// weights. A page is 16 tokens of one block.
//
// All pages that the call's requests see are laid end to end, request by request, and cut into as many equal ranges as fill
// the device with a workgroup for each of a range's KV heads (two a CU; short requests whole): a batch's longest request is
// no workgroup's alone, and lengths that a captured call only reads on the device need no bound. A workgroup of 4 waves goes through its
// range's requests; a wave takes two pages, 32 tokens, at a time and keeps references and sums of its own; the waves
// meet in LDS at a request's end. A request that a range has whole is written there, parts of others are joined by
// merge8_kernel. (One split of every request by the longest's length: 24 requests of 1000 to 8191 tokens over 8 KV heads 76
// us, ranges 63; 96 of them 243 and 201.)
//
// Memory bounds it: 256 bytes of codes a token and KV head, far above the instructions' time for any G. 64 requests of
// 8192 tokens over 8 KV heads (1.08 GB) 178 us, 6.0 TB/s; 24 of 1000 to 8191 (237 MB) 58; one of 4096 over 32 KV heads (34 MB) 15,
// of which 4 are the merge's launch. The next pages' loads ahead of a pair's products gained nothing, nor did 3 or 4 workgroups a CU.
//
// Both products run on v_mfma_f32_16x16x32_f16, for which every code and fp16 query is exact; a bf16 query row goes to fp16
// by a power of two that brings its largest value to 2^14, which leaves values down to 2^-28 of that exact. S^T =
// K q^T has 16 tokens as rows: lane l holds 16 bytes of row l % 16 at a time, two operands of 8 dimensions. Its result
// gives lane l the scores of column l % 16 (a query head) at tokens 4 (l / 16) .. + 3 of either page, which is the B
// operand of out^T = V^T P^T with that product's 32 terms in the order (l / 16, page, token). V^T's rows are the
// head's dimensions in the order 8 (l % 16) + i for the i-th of 8 products: lane l loads 8 bytes of each of its 8
// tokens, and 4x4 byte transposes (8 permutes each) make words of 4 tokens' dimension i before they become halves.
//
// Rounding: scores, references and sums are fp32. A weight enters the second product as two fp16 values, itself rounded and what
// that left, 22 bits; up to 8 query heads the lanes of the other 8 columns, whose scores are the same heads'
// again, take the second one, so that one product does. Two references are kept for that: m of the scores s for
// the sum of weights, and r of s + c for the weights of the values, each 2^7 below the largest when it was set and moved
// when that passes it by 2^15, so that neither overflows fp16 and what a value contributes keeps its bits, down to 2^-31 of the
// largest contribution to its head, whatever the blocks' exponents are (a first token with a large weight and values of 2^-40
// of the others' keeps them). Partials keep both
// references, and the result is scaled by 2^(r - m) in two steps, so values near fp32's largest stay finite.
//
// A block whose exponent says NaN makes every row NaN that sees one of its tokens. A row that sees no token is zero; one
// whose scores are all -inf is 0 / 0, NaN.
#include <algorithm>

#include "cache8.hpp"
#include "window_pages.hpp"

namespace starkv {

namespace {

constexpr int D8_THR = 256;
constexpr int D8_PART = 132;        // floats of a partial: m, sum of weights above it, r, 0, sums of values above r [128]
constexpr int D8_MAX_GROUP = 16;    // query heads per KV head: the columns of a matrix product
constexpr float D8_LEAST = -3.402823466e38f;  // the reference of tokens whose scores are all -inf

// Calls of more pages (a KV head's, 4 KB of codes) load keys past the caches: 64 x 8192 tokens of 8 heads 193 -> 178 us, 24 x 8192
// 84 -> 80, 8 x 8192 (134 MB) 37 -> 33; keys and values both past them 180, 83, 36. Fewer pages may be in the last level
// (256 MB) from the step before: 4 x 8192 (67 MB) 21.8 us, 23.7 past it.
constexpr int D8_ONCE = (96 << 20) / 4096;

// A short request costs a range its latencies (look-up, rows, the waves' meeting: about 4 us) more than its pages, so
// one of up to half as much again as a range's pages, 16 at most, is the whole of the range's that has its first page: 64 requests
// of 20 to 60 tokens over 8 KV heads 20.9 -> 14.6 us, of 100 to 200 23.1 -> 19.2 (up to 8 pages 24.1); always up to 16 pages, 8
// requests of 200 to 900 took 15.8 and not 13.9.
constexpr int D8_WHOLE = 16;

// Where a call's requests have no more than 16 pages each on average, it is cut into up to four times as many ranges, one
// a request: 200 requests of 20 to 60 tokens over 8 KV heads 32.3 -> 27.5 us, 256 of 100 to 200 44.9 -> 42.1. Longer ones gain
// nothing (256 of 300 to 700: 83.8 and 84.1) and would be cut more often.
constexpr int D8_MORE = 4;

struct Decode8Params {
    const uint16_t* q; int64_t q_s0, q_s1;                              // elements
    const uint8_t* kc; const uint8_t* vc; int64_t c_s0, c_s1, c_s2;     // bytes
    const int8_t* ex; int64_t x_s0, x_s1;                               // [num_blocks][Hkv][2]
    int bs_shift; int64_t num_blocks;                                   // block_size = 16 << bs_shift
    const int32_t* bt; int64_t bt_s0, bt_s1;
    const int32_t* seq_lens; int span;                                  // lengths are clamped to span
    int n, Hkv, G, ranges, base, window, sinks;                         // base: the ranges of long requests
    float sc;                                                           // scale * log2(e)
    int2* where;                                                        // [n]: first range, ranges
    float* part;                                                        // [ranges][2][H][D8_PART]
    uint16_t* out; int64_t o_s0, o_s1;
};

__device__ __forceinline__ SeenPages seen_by(const Decode8Params& p, int b) {
    return seen_pages(min(max(p.seq_lens[b], 0), p.span), p.window, p.sinks);
}

__device__ __forceinline__ int scan_wave(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}

// A range of the call's pages, request by request: its first page's request and place there, and its length. All
// waves find it by themselves: a lane counts the pages of n / 64 requests, then of one in the lane's that has the first.
struct Range8 {
    int b, k, left, per, whole;  // per: pages a range; whole: up to which one range takes all of a request
    bool once;            // keys go past the caches
};

__device__ __forceinline__ Range8 find_range(const Decode8Params& p, int range) {
    const int lane = threadIdx.x & 63, some = (p.n + 63) >> 6;
    int own = 0, end;
    if (p.n == 1) {
        own = end = seen_by(p, 0).pages;
    } else {
        for (int b = lane * some; b < min((lane + 1) * some, p.n); ++b) own += seen_by(p, b).pages;
        end = scan_wave(own);
    }
    const int total = __builtin_amdgcn_readlane(end, 63);
    Range8 g;
    const int ranges = total <= 16 * p.n ? p.ranges : min(p.base, p.ranges);
    // At least two pages a wave of a long request; of short ones about one request (6 requests of one token over 8 KV heads
    // in one range took 28 us, in six 8.4).
    g.per = max((total + ranges - 1) / ranges, max(min(total / p.n, 8), 1));
    g.whole = min(g.per + (g.per + 1) / 2, D8_WHOLE);
    g.once = (int64_t)total * p.Hkv > D8_ONCE;
    g.b = g.k = 0;
    // Where the ranges are enough for that, each has pages of one request only, since a range's second request costs as
    // much time as its first: 24 requests of 30 to 300 tokens over 8 KV heads 19.6 -> 13.9 us, 64 of 100 to 200 19.0 -> 14.7, 4 of 200
    // to 4000 over 4 18.5 -> 14.8. Not looked into for more requests than the device has room for (200 of 20 to 60: 27.5, with
    // it 29.1).
    const auto parts = [&](int pages) { return pages <= g.whole ? (int)(pages > 0) : (pages + g.per - 1) / g.per; };
    bool apart = false;
    int start = range * g.per;
    g.left = min(g.per, total - start);
    if (p.n > 1 && p.n <= p.base && (total <= 16 * p.n || total < 8 * ranges)) {
        int own1 = 0;
        if (some == 1)
            own1 = parts(own);
        else
            for (int b = lane * some; b < min((lane + 1) * some, p.n); ++b) own1 += parts(seen_by(p, b).pages);
        const int end1 = scan_wave(own1), need = __builtin_amdgcn_readlane(end1, 63);
        if (need <= ranges) {
            apart = true;
            own = own1;
            end = end1;
            start = range;
            g.left = need - range;
        }
    }
    if (g.left <= 0) return g;
    int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= start));
    if (some > 1) {
        start -= __builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(own, at);
        const int b1 = min((at + 1) * some, p.n);
        for (g.b = at * some;; g.b += 64) {
            own = g.b + lane < b1 ? seen_by(p, g.b + lane).pages : 0;
            if (apart) own = parts(own);
            end = scan_wave(own);
            at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= start));
            if (at < 64) break;
            start -= __builtin_amdgcn_readlane(end, 63);
        }
    }
    g.b += at;
    const int size = __builtin_amdgcn_readlane(own, at);
    g.k = start - __builtin_amdgcn_readlane(end, at) + size;
    if (apart) {
        const int pages = seen_by(p, g.b).pages;
        g.k *= g.per;
        g.left = pages <= g.whole ? pages : min(g.per, pages - g.k);
    } else if (g.k > 0 && size <= g.whole) {  // the range before has it
        g.left -= size - g.k;
        g.k = 0;
        if (g.left > 0)
            do ++g.b;
            while (seen_by(p, g.b).pages == 0);
    }
    return g;
}

// The end of what a range with `left` pages to its end takes of a request from page k on.
__device__ __forceinline__ int taken(const Range8& g, const SeenPages& seen, int k, int left) {
    return seen.pages <= g.whole ? seen.pages : min(seen.pages, k + left);
}

__device__ __forceinline__ f32x4_t mfma_f16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Two floats to fp16, packed, and what the rounding left of them.
__device__ __forceinline__ uint32_t split_half(float& a, float& b) {
    const _Float16 x = (_Float16)a, y = (_Float16)b;
    a -= (float)x;
    b -= (float)y;
    return (uint32_t)__builtin_bit_cast(uint16_t, x) | (uint32_t)__builtin_bit_cast(uint16_t, y) << 16;
}

// Words of 4 dimensions of tokens 0 .. 3 to words of 4 tokens of dimensions 0 .. 3.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// The result of sums a above reference r and l above m: a / l 2^(r - m), in two steps, of which 2^(r - m) may be past fp32's
// range where the result is not. 0 where there were no tokens.
__device__ __forceinline__ float weigh_out(float a, float l, float m, float r) {
    const float half = exp2f(0.5f * (r - m));
    return m == -INFINITY ? 0.f : a / l * half * half;
}

// What a wave's lanes know of 32 pairs of pages: pages c0, c0 + 1, c0 + 8, c0 + 9, ... of the request's. The block, the places
// that are seen | the page's place in the block << 16, the exponents (which the rows need not wait for).
struct Look8 {
    int blk, ek, ev;
    uint32_t see;
};

__device__ __forceinline__ Look8 look_up(const Decode8Params& p, const SeenPages& seen, int b, int h, int c0, int k1) {
    const int lane = threadIdx.x & 63, mine = c0 + 8 * (lane >> 1) + (lane & 1);
    Look8 l = {0, 0, 0, 0};
    if (mine < k1) {
        const int pg = seen.page(mine);
        l.blk = p.bt[b * p.bt_s0 + (pg >> p.bs_shift) * p.bt_s1];
        l.see = seen.mask(pg) | (uint32_t)(pg & ((1 << p.bs_shift) - 1)) << 16;
        if (l.blk < 0 || l.blk >= p.num_blocks) l.blk = l.see = 0;  // no block of the cache: no tokens
        const int8_t* e = p.ex + l.blk * p.x_s0 + h * p.x_s1;
        l.ek = e[0];
        l.ev = e[1];
    }
    return l;
}

// A KV head's part of a range, from the block index: request by request, the result of its query heads where the range has
// all of a request's pages, else a partial. What lies where and the queries of the next request are on their way while
// the waves of one meet. MANY: 9 to 16 query heads.
template <int CT, int QDT, bool MANY>
__global__ __launch_bounds__(D8_THR, 3) void decode8_kernel(const Decode8Params p) {
    extern __shared__ float s_dyn[];  // [4 waves][G][D8_PART] for the merge
    const int range = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, H = p.Hkv * p.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = MANY ? lane & 15 : lane & 7, quad = lane >> 4;  // the lane's query head
    if (p.ranges == 1)  // no merge follows, which writes the rows that see no token
        for (int b = 0; b < p.n; ++b)
            if (seen_by(p, b).pages == 0)
                for (int i = tid; i < p.G * 128; i += D8_THR)
                    store_f(p.out, b * p.o_s0 + (h * p.G + (i >> 7)) * p.o_s1 + (i & 127), QDT, 0.f);
    const Range8 g = find_range(p, range);
    if (g.left <= 0) return;
    const uint8_t* kh = p.kc + h * p.c_s2 + 16 * quad + (int64_t)(lane & 15) * p.c_s1;
    const uint8_t* vh = p.vc + h * p.c_s2 + 8 * (lane & 15) + (int64_t)(4 * quad) * p.c_s1;
    // The head's row: dimensions 64 st + 16 quad .. + 15, two operands.
    uint4 w[2][2];
    const auto load_q = [&](int b) {
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                w[st][x] = col < p.G ? *(const uint4*)(p.q + b * p.q_s0 + (int64_t)(h * p.G + col) * p.q_s1 + 64 * st + 16 * quad + 8 * x)
                                     : make_uint4(0, 0, 0, 0);
    };
    int b = g.b, k0 = g.k, left = g.left;
    SeenPages seen = seen_by(p, b);
    int k1 = taken(g, seen, k0, left);
    Look8 ahead = look_up(p, seen, b, h, k0 + 2 * wave, k1);
    load_q(b);
    for (;;) {
        const bool whole = k0 == 0 && k1 == seen.pages;
        if (h == 0 && k0 == 0 && tid == 0) p.where[b] = make_int2(range, 1 + (seen.pages - k1 + g.per - 1) / g.per);
        uint4 qf[2][2];  // fp16 values of the queries, times 2^up
        int up_q = 0;
        if constexpr (QDT == STARKV_F16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[i >> 1][i & 1] = w[i >> 1][i & 1];
        } else {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t v = ((const uint32_t*)&w[i >> 1][i & 1])[k];
                    top = fmaxf(top, fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xffff0000u))));
                }
            top = max_rows(top);
            // 2^14 <= top 2^up < 2^15; of zeros, subnormal numbers and infinities the nearest power there is.
            up_q = min(max(141 - (int)(__float_as_uint(top) >> 23), -126), 126);
            const float by = __uint_as_float((uint32_t)(up_q + 127) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                half8_t o;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t v = ((const uint32_t*)&w[i >> 1][i & 1])[k];
                    o[2 * k] = (_Float16)(__uint_as_float(v << 16) * by);
                    o[2 * k + 1] = (_Float16)(__uint_as_float(v & 0xffff0000u) * by);
                }
                qf[i >> 1][i & 1] = __builtin_bit_cast(uint4, o);
            }
        }
        float m = -INFINITY, r = -INFINITY, l = 0.f;
        f32x4_t acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        // A wave takes pages k0 + 2 wave and the next, k0 + 2 wave + 8 and the next, ..., 32 such pairs' places at a time in its
        // lanes: what lies where, which places are seen and the exponents, which the rows need not wait for.
        for (int c0 = k0 + 2 * wave; c0 < k1; c0 += 8 * 32) {
            const Look8 now = c0 < k0 + 8 ? ahead : look_up(p, seen, b, h, c0, k1);
            const int pairs = min((k1 - c0 + 7) / 8, 32);
            for (int i = 0; i < pairs; ++i) {
                uint32_t see[2];
                int at[2], place[2], ek[2], ev[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    at[x] = __builtin_amdgcn_readlane(now.blk, 2 * i + x);
                    const uint32_t v = (uint32_t)__builtin_amdgcn_readlane((int)now.see, 2 * i + x);
                    place[x] = (int)(v >> 16);
                    see[x] = v & 0xffffu;
                }
                if ((see[0] | see[1]) == 0) continue;
                uint4 kr[2][2];
                uint2 vr[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    // A page of which nothing is seen reads the other one again. A page lies within its block whatever
                    // the request's length, so every row of it can be read.
                    const int y = see[x] ? x : x ^ 1;
                    const int64_t base = at[y] * p.c_s0 + (int64_t)(16 * place[y]) * p.c_s1;
                    if (g.once) {
#pragma unroll
                        for (int st = 0; st < 2; ++st) kr[x][st] = load_once16(kh + base + 64 * st);
                    } else {
#pragma unroll
                        for (int st = 0; st < 2; ++st) kr[x][st] = *(const uint4*)(kh + base + 64 * st);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) vr[x][j] = *(const uint2*)(vh + base + j * p.c_s1);
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    ek[x] = __builtin_amdgcn_readlane(now.ek, 2 * i + x);
                    ev[x] = __builtin_amdgcn_readlane(now.ev, 2 * i + x);
                }
                float sv[2][4], up[2];  // scores; the exponents of the values
                float mx = -INFINITY, rx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const uint2 a = c8_halves<CT>(kr[x][st].x), c = c8_halves<CT>(kr[x][st].y);
                        const uint2 e = c8_halves<CT>(kr[x][st].z), f = c8_halves<CT>(kr[x][st].w);
                        d = mfma_f16(make_uint4(a.x, a.y, c.x, c.y), qf[st][0], d);
                        d = mfma_f16(make_uint4(e.x, e.y, f.x, f.y), qf[st][1], d);
                    }
                    const float sc = ek[x] == C8_NAN ? __builtin_nanf("") : p.sc;
                    up[x] = ev[x] == C8_NAN && see[x] != 0 ? __builtin_nanf("") : (float)ev[x];
#pragma unroll
                    for (int k = 0; k < 4; ++k) sv[x][k] = __builtin_ldexpf(d[k] * sc, ek[x] - up_q);  // whatever the two exponents are
                    if (see[x] != 0xffffu) {  // tokens out of sight: no score, and codes of 0 (an e4m3 code may be NaN)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const bool ok = see[x] >> (4 * quad + k) & 1u;
                            sv[x][k] = ok ? sv[x][k] : -INFINITY;
                            vr[x][k] = ok ? vr[x][k] : make_uint2(0, 0);
                        }
                    }
                    const float px = fmaxf(fmaxf(sv[x][0], sv[x][1]), fmaxf(sv[x][2], sv[x][3]));
                    mx = fmaxf(mx, px);
                    rx = fmaxf(rx, px + up[x]);
                }
                mx = max_rows(mx);
                rx = max_rows(rx);
                m = fmaxf(m, D8_LEAST);
                r = fmaxf(r, D8_LEAST);
                if (__builtin_amdgcn_ballot_w64(mx > m + 15.f || rx > r + 15.f) != 0) {
                    const float mn = mx > m + 15.f ? mx - 7.f : m, rn = rx > r + 15.f ? rx - 7.f : r;
                    l *= mn == m ? 1.f : exp2f(m - mn);
                    const float alpha = rn == r ? 1.f : exp2f(r - rn);
                    m = mn;
                    r = rn;
#pragma unroll
                    for (int i8 = 0; i8 < 8; ++i8) acc[i8] *= alpha;
                }
                float pe[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float e = up[x] + (m - r), f = exp2f(e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool ok = see[x] >> (4 * quad + k) & 1u;
                        const float w = ok ? exp2f(sv[x][k] - m) : 0.f;
                        l += w;
                        pe[x][k] = ok ? w * f : 0.f;
                    }
                    // Values so much larger than others' that a weight of next to nothing counts: past fp32's range one by one.
                    if (__builtin_amdgcn_ballot_w64(e > 60.f) != 0) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) pe[x][k] = see[x] >> (4 * quad + k) & 1u ? exp2f(sv[x][k] + (up[x] - r)) : 0.f;
                    }
                }
                // The weights' values: the first, and what it left; up to 8 heads the lanes of the second columns take that.
                uint4 pw[MANY ? 2 : 1];
                pw[0] = make_uint4(split_half(pe[0][0], pe[0][1]), split_half(pe[0][2], pe[0][3]),
                                   split_half(pe[1][0], pe[1][1]), split_half(pe[1][2], pe[1][3]));
                const uint4 rest = make_uint4(split_half(pe[0][0], pe[0][1]), split_half(pe[0][2], pe[0][3]),
                                              split_half(pe[1][0], pe[1][1]), split_half(pe[1][2], pe[1][3]));
                if constexpr (MANY) {
                    pw[1] = rest;
                } else if (lane & 8) {
                    pw[0] = rest;
                }
#pragma unroll
                for (int hd = 0; hd < 2; ++hd) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[x][j] = hd ? vr[x][j].y : vr[x][j].x;
                        transpose4(w[x]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 a = c8_halves<CT>(w[0][i]), c = c8_halves<CT>(w[1][i]);
                        const uint4 vt = make_uint4(a.x, a.y, c.x, c.y);
#pragma unroll
                        for (int k = 0; k < (MANY ? 2 : 1); ++k) acc[4 * hd + i] = mfma_f16(vt, pw[k], acc[4 * hd + i]);
                    }
                }
            }
        }
        left -= k1 - k0;
        int next = b;
        SeenPages then = seen;
        if (left > 0) {
            do then = seen_by(p, ++next);
            while (then.pages == 0);
            ahead = look_up(p, then, next, h, 2 * wave, taken(g, then, 0, left));
            load_q(next);
        }
        l = sum_rows(l);
        if constexpr (!MANY) {  // both columns of a head: lanes 8 apart in a row of 16
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[i8][x] += dpp_f<0x128>(acc[i8][x]);  // row_ror:8
        }
        __syncthreads();  // the request before is done with s_dyn
        if (col < p.G && (MANY || !(lane & 8))) {
            float* w = s_dyn + (wave * p.G + col) * D8_PART;
            if (quad == 0) *(float4*)w = make_float4(m, l, r, 0.f);
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // dimensions 32 quad + 8 x + i
                *(float4*)(w + 4 + 32 * quad + 8 * x) = make_float4(acc[0][x], acc[1][x], acc[2][x], acc[3][x]);
                *(float4*)(w + 8 + 32 * quad + 8 * x) = make_float4(acc[4][x], acc[5][x], acc[6][x], acc[7][x]);
            }
        }
        __syncthreads();
        for (int i = tid; i < p.G * 128; i += D8_THR) {
            const int g = i >> 7, d = i & 127;
            const float* w = s_dyn + g * D8_PART;
            float M = -INFINITY, R = -INFINITY, lt = 0.f, a = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                M = fmaxf(M, w[k * p.G * D8_PART]);
                R = fmaxf(R, w[k * p.G * D8_PART + 2]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float* x = w + k * p.G * D8_PART;
                // A wave without tokens has references of -inf and sums of 0.
                lt = fmaf(x[1], x[0] == -INFINITY ? 1.f : exp2f(x[0] - M), lt);
                a = fmaf(x[4 + d], x[2] == -INFINITY ? 1.f : exp2f(x[2] - R), a);
            }
            const int hq = h * p.G + g;
            if (whole) {
                store_f(p.out, b * p.o_s0 + hq * p.o_s1 + d, QDT, weigh_out(a, lt, M, R));
            } else {
                float* pp = p.part + ((int64_t)(2 * range + (k0 == 0)) * H + hq) * D8_PART;
                if (d == 0) *(float4*)pp = make_float4(M, lt, R, 0.f);
                pp[4 + d] = a;
            }
        }
        if (left <= 0) break;
        b = next;
        seen = then;
        k0 = 0;
        k1 = taken(g, seen, 0, left);
    }
}

// A head's partials joined by WAVES waves: sums of weights above the largest m, of values above the largest r. The first lies
// second in its range (other requests may end there), the others first in theirs. A wave takes a run of them; its lane s of
// 64 holds the factors of 64 partials at a time and sums dimensions 2 s and 2 s + 1, eight partials' loads in flight.
template <int QDT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void merge8_kernel(const Decode8Params p) {
    __shared__ float4 s_ref[WAVES];
    __shared__ float2 s_sum[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hq = blockIdx.x, b = blockIdx.y, H = p.Hkv * p.G;
    const int64_t to = b * p.o_s0 + hq * p.o_s1 + 2 * lane;
    const int2 where = p.where[b];
    if (seen_by(p, b).pages == 0) {  // no workgroup has it, nor has one said where it is
        if (wave == 0) {
            store_f(p.out, to, QDT, 0.f);
            store_f(p.out, to + 1, QDT, 0.f);
        }
        return;
    }
    if (where.y == 1) return;
    const auto part = [&](int s) { return p.part + ((int64_t)(2 * (where.x + s) + (s == 0)) * H + hq) * D8_PART; };
    const int run = (where.y + WAVES - 1) / WAVES, end = min((wave + 1) * run, where.y);
    float M = -INFINITY, R = -INFINITY, lt = 0.f;
    float2 a = make_float2(0.f, 0.f);
    for (int c0 = wave * run; c0 < end; c0 += 64) {
        const int count = min(end - c0, 64);
        float2 v[8];  // the first eight's sums are on their way with the references
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = *(const float2*)(part(c0 + min(u, count - 1)) + 4 + 2 * lane);
        const float4 mine = *(const float4*)part(c0 + min(lane, count - 1));
        const float m = lane < count ? mine.x : -INFINITY, r = lane < count ? mine.z : -INFINITY;
        const float M1 = fmaxf(M, wave_max(m)), R1 = fmaxf(R, wave_max(r));
        // A partial without tokens has references of -inf and sums of 0.
        const float fl = m == -INFINITY ? 0.f : mine.y * exp2f(m - M1), fa = r == -INFINITY ? 0.f : exp2f(r - R1);
        const float before = R == -INFINITY ? 0.f : exp2f(R - R1);
        lt = fmaf(lt, M == -INFINITY ? 0.f : exp2f(M - M1), wave_sum(fl));
        a.x *= before;
        a.y *= before;
        M = M1;
        R = R1;
        for (int s0 = 0; s0 < count; s0 += 8) {
            if (s0 > 0) {
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = *(const float2*)(part(c0 + min(s0 + u, count - 1)) + 4 + 2 * lane);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(fa), (s0 + u) & 63));
                if (s0 + u < count) {
                    a.x = fmaf(v[u].x, fs, a.x);
                    a.y = fmaf(v[u].y, fs, a.y);
                }
            }
        }
    }
    if constexpr (WAVES > 1) {
        if (lane == 0) s_ref[wave] = make_float4(M, lt, R, 0.f);
        s_sum[wave][lane] = a;
        __syncthreads();
        if (wave > 0) return;
        float4 x[WAVES];
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            x[k] = s_ref[k];
            M = fmaxf(M, x[k].x);
            R = fmaxf(R, x[k].z);
        }
        lt = a.x = a.y = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float f = x[k].z == -INFINITY ? 0.f : exp2f(x[k].z - R);
            const float2 v = s_sum[k][lane];
            lt = fmaf(x[k].y, x[k].x == -INFINITY ? 0.f : exp2f(x[k].x - M), lt);
            a.x = fmaf(v.x, f, a.x);
            a.y = fmaf(v.y, f, a.y);
        }
    }
    store_f(p.out, to, QDT, weigh_out(a.x, lt, M, R));
    store_f(p.out, to + 1, QDT, weigh_out(a.y, lt, M, R));
}

int decode8_base(int num_kv_heads) { return std::max(1, 2 * device_cus() / num_kv_heads); }

// Ranges that a call's pages are cut into, at most: workgroups for 2 a CU with a range's KV heads, more for many requests.
int decode8_ranges(int n, int num_kv_heads, int span, int window, int sinks) {
    const int64_t pages = (int64_t)n * seen_pages_most(span, window, sinks);
    if (n == 1) return (int)std::min<int64_t>(decode8_base(num_kv_heads), pages <= D8_WHOLE ? 1 : (pages + 7) / 8);
    const int base = decode8_base(num_kv_heads);
    return (int)std::min<int64_t>(std::max(base, std::min(n, D8_MORE * base)), pages);
}

size_t decode8_bytes(int n, int num_heads, int ranges) {
    return (((size_t)n * sizeof(int2) + 255) & ~(size_t)255) + (size_t)ranges * 2 * num_heads * D8_PART * 4;
}

template <int CT, int QDT>
const void* decode_pick(int G) {
    return G <= 8 ? (const void*)&decode8_kernel<CT, QDT, false> : (const void*)&decode8_kernel<CT, QDT, true>;
}

template <int QDT>
const void* merge_pick(int waves) {
    return waves == 1 ? (const void*)&merge8_kernel<QDT, 1> : waves == 4 ? (const void*)&merge8_kernel<QDT, 4> : (const void*)&merge8_kernel<QDT, 16>;
}

}  // namespace

}  // namespace starkv

using namespace starkv;

extern "C" {

size_t starkv_decode_kv8_workspace_bytes(int n, int num_heads, int num_kv_heads, int max_seq_len, int window, int sinks) {
    if (n < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || max_seq_len < 1 || window < 0 || sinks < 0) return 256;
    return decode8_bytes(n, num_heads, decode8_ranges(n, num_kv_heads, max_seq_len, window, sinks));
}

int starkv_decode_kv8(void* stream, const void* query, int64_t q_s0, int64_t q_s1, int dtype, const void* k_codes,
                      const void* v_codes, int64_t c_s0, int64_t c_s1, int64_t c_s2, int code_type,
                      const int8_t* exponents, int64_t x_s0, int64_t x_s1, int block_size, int64_t num_blocks,
                      const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width, const int32_t* seq_lens,
                      int n, int num_heads, int num_kv_heads, int max_seq_len, int window, int sinks, float scale,
                      void* out, int64_t o_s0, int64_t o_s1, void* workspace, size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && max_seq_len >= 1, "decode_kv8: n=%d (up to 65535) max_seq_len=%d", n, max_seq_len);
    SKV_CHECK(window >= 0 && sinks >= 0, "decode_kv8: window=%d sinks=%d", window, sinks);
    if (n == 0) return STARKV_OK;
    SKV_CHECK(query && k_codes && v_codes && exponents && block_table && seq_lens && out && workspace, "decode_kv8: null pointer");
    SKV_CHECK(num_kv_heads >= 1 && num_heads >= num_kv_heads && num_heads % num_kv_heads == 0 &&
                  num_heads / num_kv_heads <= D8_MAX_GROUP,
              "decode_kv8: %d query heads over %d KV heads (1 to 16 each)", num_heads, num_kv_heads);
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "decode_kv8: queries must be bf16 or fp16");
    SKV_CHECK(code_type == STARKV_I8 || code_type == STARKV_E4M3, "decode_kv8: codes must be int8 or e4m3");
    SKV_CHECK(c8_block_shift(block_size) >= 0, "decode_kv8: block_size must be 16 times a power of two, at most %d", C8_MAX_BLOCK);
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff && bt_width >= 1, "decode_kv8: empty cache or block table");
    SKV_CHECK(((uintptr_t)query | (uintptr_t)k_codes | (uintptr_t)v_codes) % 16 == 0 && (q_s0 | q_s1) % 8 == 0 &&
                  (c_s0 | c_s1 | c_s2) % 16 == 0 && (uintptr_t)workspace % 16 == 0,
              "decode_kv8: rows must be 16-byte aligned");
    const size_t need = starkv_decode_kv8_workspace_bytes(n, num_heads, num_kv_heads, max_seq_len, window, sinks);
    SKV_CHECK(workspace_bytes >= need, "decode_kv8: workspace %zu bytes < %zu", workspace_bytes, need);
    Decode8Params p;
    p.q = (const uint16_t*)query; p.q_s0 = q_s0; p.q_s1 = q_s1;
    p.kc = (const uint8_t*)k_codes; p.vc = (const uint8_t*)v_codes;
    p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.ex = exponents; p.x_s0 = x_s0; p.x_s1 = x_s1;
    p.bs_shift = c8_block_shift(block_size) - 4; p.num_blocks = num_blocks;
    p.bt = block_table; p.bt_s0 = bt_s0; p.bt_s1 = bt_s1;
    p.seq_lens = seq_lens;
    p.span = (int)std::min<int64_t>({(int64_t)bt_width * block_size, 0x7ffffff0, (int64_t)max_seq_len});
    p.n = n; p.Hkv = num_kv_heads; p.G = num_heads / num_kv_heads;
    p.base = decode8_base(num_kv_heads);
    p.ranges = decode8_ranges(n, num_kv_heads, max_seq_len, window, sinks);
    p.window = window; p.sinks = sinks;
    p.sc = scale * 1.4426950408889634f;
    p.where = (int2*)workspace;
    p.part = (float*)((char*)workspace + (((size_t)n * sizeof(int2) + 255) & ~(size_t)255));
    p.out = (uint16_t*)out; p.o_s0 = o_s0; p.o_s1 = o_s1;
    SKV_CHECK((int64_t)n * seen_pages_most(p.span, window, sinks) < 1ll << 30,  // a range's first page stays in 32 bits
              "decode_kv8: %d requests of up to %d tokens in one call", n, p.span);
    SKV_CHECK(num_heads <= 65535, "decode_kv8: %d heads", num_heads);
    const bool bf = dtype == STARKV_BF16;
    const void* fn = code_type == STARKV_I8 ? bf ? decode_pick<STARKV_I8, STARKV_BF16>(p.G) : decode_pick<STARKV_I8, STARKV_F16>(p.G)
                                            : bf ? decode_pick<STARKV_E4M3, STARKV_BF16>(p.G) : decode_pick<STARKV_E4M3, STARKV_F16>(p.G);
    void* args[] = {(void*)&p};
    SKV_HIP(hipLaunchKernel(fn, dim3((unsigned)((int64_t)p.ranges * num_kv_heads)), dim3(D8_THR), args,
                            (size_t)4 * p.G * D8_PART * 4, (hipStream_t)stream));
    if (p.ranges == 1) return STARKV_OK;
    // One wave joins eight partials in the time of one; more by several: one request of 8192 tokens over 8 KV heads (64) 17.6 us by
    // one wave, 14.4 by 4, 15.1 by 16; of 65536 over one (512) 58.7, 24.6, 18.1; of 1000 over 8 (8) 9.7 by one, 10.3 by 4.
    const int waves = p.ranges < 16 * n ? 1 : p.ranges < 128 * n ? 4 : 16;
    SKV_HIP(hipLaunchKernel(bf ? merge_pick<STARKV_BF16>(waves) : merge_pick<STARKV_F16>(waves), dim3(num_heads, n), dim3(64 * waves),
                            args, 0, (hipStream_t)stream));
    return STARKV_OK;
}

}  // extern "C"
