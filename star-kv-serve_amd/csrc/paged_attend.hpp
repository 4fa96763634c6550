// One token's attention over pages of an uncompressed paged cache, on matrix instructions: the body
// that the decode over selected blocks (sparse_decode.hip), the decode that weighs its tokens
// (evict.hip) and the one through a window (window_decode.hip) share.
//
// For a request b, a KV head h and its G <= 16 query heads: s_g(t) = scale log2(e) q_g . k_t over the
// tokens t of the unit's pages, p = 2^(s - m), out_g = sum p v / sum p. A page is 16 tokens of one
// block. A workgroup of 4 waves takes a range of the unit's pages (a split); a wave takes two pages,
// 32 tokens, at a time and keeps its own running reference m and sums; the waves meet in LDS at the
// end, the splits in attend_merge_kernel.
//
// Both products run on v_mfma_f32_16x16x32 with nothing but registers between memory and the matrix
// unit: S^T = K q^T takes 16 tokens as rows, so a lane holds row l % 16 of the page's keys as they lie
// in memory (64 bytes of each of 16 rows a load) and the 16 columns are the query heads. The result
// gives lane l the scores of column l % 16 at tokens 4 (l / 16) .. + 3 of either page, which is the B
// operand of out^T = V^T P^T with the product's 32 terms in the order (l / 16, page, token): P goes
// from one product into the other in place. V^T's rows are the head's dimensions in the order
// 8 (l % 16) + i for the i-th of 8 products, so the A operand is dimension i of the 16 bytes that lane
// l loaded of each of its 8 tokens (4 rows of 256 bytes a load), gathered with 4 byte permutes. A lane
// ends with 32 consecutive dimensions of one column.
//
// Memory bounds it: 512 bytes of keys and values a token and KV head, far above the instructions' time for
// any G. 32 requests of up to 2048 selected tokens over 32 KV heads (1.07 GB) 189 us, 5.7 TB/s; 24 of 1000
// to 8191 tokens over 8 KV heads with their scores left behind (445 MB) 97. The next tile's loads ahead of a
// tile's products gained nothing (189 -> 193, at half the waves), nor did loads past the caches.
//
// Rounding: scores, references and sums are fp32. The weights enter the second product as three values
// of the cache's type, the weight in it, what that left and what that left: all 24 bits of a bf16 weight
// (each value cut) and of an fp16 one (rounded) down to 2^-24, where fp16 ends. Up to 8 query heads the second and
// third values take the other 8 columns, whose scores are the same heads' again, so that two products do; 9 to 16
// heads take a product each. Two values, 16 bits of a bf16 weight, made results low by up to 2^-15 and were
// 1 % faster at most. The reference lies 2^7 below the largest score seen when it was set and moves when a score
// passes it by 2^15 (fp16 weights stay finite, and small ones keep 22 bits of range above its subnormals).
//
// A wave that has seen tokens has a finite reference or +inf: scores of -inf (an infinite key) weigh 0 against it,
// and where a row has no others its sums are 0 and the result 0 / 0. A reference of -inf says that there were no
// tokens, whose result is 0.
//
// An infinite value times a weight's second or third value would be NaN or an infinity of the other sign where that
// is 0 or negative. A workgroup whose sums are not finite though its weights are goes over its pages once more, the finite
// values as before and the others times 1 where their token's weight is not 0: what the weight's bits are no
// longer matters. Finite values pay for the look at the sums alone (32 requests 190 us with and without it, one
// request of 4096 tokens 17.4 -> 17.8).
#pragma once

#include <algorithm>

#include "common.hpp"
#include "window_pages.hpp"

namespace starkv {

constexpr int AT_THR = 256;
constexpr int AT_CHUNK = 512;      // pages whose places are looked up at a time
constexpr int AT_PART = 132;       // floats of a partial: reference, sum of weights, 0, 0, out[128]
constexpr int AT_MAX_SPLITS = 128;
constexpr int AT_MAX_GROUP = 16;   // query heads per KV head: the columns of a matrix product
constexpr float AT_LOG2E = 1.4426950408889634f;
// What weights are multiplied by. bf16 values reach fp32's largest: times weights of 2^15 and summed, those past 2^100 or
// so left it. fp16 values are far from it, and fp16 weights have no such range.
template <int DT>
constexpr float AT_DOWN = DT == STARKV_BF16 ? 0x1p-40f : 1.f;
constexpr float AT_LEAST = -3.402823466e38f;  // the reference of tokens whose scores are all -inf

// Which pages a unit has: all of its request, with the scores left behind; those of selected blocks; those seen
// through a window.
enum { AT_SCORES, AT_SPARSE, AT_WINDOW };

struct AttendParams {
    const uint16_t* q; int64_t q_s0, q_s1;                               // elements, as all strides here
    const uint16_t* kc; const uint16_t* vc; int64_t c_s0, c_s1, c_s2;
    int bs_shift; int64_t num_blocks;                                    // block_size = 16 << bs_shift
    const int32_t* bt; int64_t bt_s0, bt_s1;
    const int32_t* seq_lens; int span;                                   // lengths are clamped to span
    int n, Hkv, G, splits, pps;                                          // pps: pages per split
    float sc;                                                            // scale * log2(e)
    const int32_t* sel; int64_t sel_s0, sel_s1; int keep;                // SPARSE: logical blocks [n][Hkv][keep]
    float* lg; int64_t lg_row;                                           // SCORES: [n][Hkv][page][G][16], lg_row a unit
    int window, sinks;                                                   // WINDOW
    float* part;                                                         // [n][H][splits][AT_PART]
    uint16_t* out; int64_t o_s0, o_s1;
};

__device__ __forceinline__ int attend_length(const AttendParams& p, int b) {
    return min(max(p.seq_lens[b], 0), p.span);
}

template <int DT>
__device__ __forceinline__ f32x4_t attend_mfma(uint4 a, uint4 b, f32x4_t c) {
    if constexpr (DT == STARKV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
}

// Two values in DT, packed, and as they became: bf16 by its upper bits (what they leave goes into the second
// product too), fp16 to the nearest (its subnormals leave nothing).
template <int DT>
__device__ __forceinline__ uint32_t attend_pack(float a, float b, float& ra, float& rb) {
    if constexpr (DT == STARKV_BF16) {
        ra = __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        rb = __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    } else {
        const _Float16 lo = (_Float16)a, hi = (_Float16)b;
        ra = (float)lo;
        rb = (float)hi;
        return (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
    }
}

// Four weights packed, and `own` of that taken off them: all of it or nothing.
template <int DT>
__device__ __forceinline__ uint2 attend_take(float (&p)[4], float own) {
    float r[4];
    const uint2 v = make_uint2(attend_pack<DT>(p[0], p[1], r[0], r[1]), attend_pack<DT>(p[2], p[3], r[2], r[3]));
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = fmaf(-own, r[i], p[i]);
    return v;
}

// The halves of a word that hold infinities or NaN.
template <int DT>
__device__ __forceinline__ uint32_t attend_odd(uint32_t w) {
    const uint32_t top = DT == STARKV_BF16 ? 0x7f80u : 0x7c00u, x = w & 0x7fff7fffu;
    return (x >> 16 >= top ? 0xffff0000u : 0) | ((x & 0xffffu) >= top ? 0xffffu : 0);
}

// 1 for each of two weights that is not 0, packed.
template <int DT>
__device__ __forceinline__ uint32_t attend_ones(float a, float b) {
    const uint32_t one = DT == STARKV_BF16 ? 0x3f80u : 0x3c00u;
    return (a > 0.f ? one : 0) | (b > 0.f ? one << 16 : 0);
}

// Component i of a 16-byte register row.
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Dimension i of 8 of a lane's 8 tokens, in the order of the second product's terms.
__device__ __forceinline__ uint4 attend_column(const uint4 (&v)[2][4], int i) {
    const uint32_t pick = i & 1 ? 0x07060302u : 0x05040100u;  // both high halves, or both low ones
    return make_uint4(__builtin_amdgcn_perm(word_of(v[0][1], i >> 1), word_of(v[0][0], i >> 1), pick),
                      __builtin_amdgcn_perm(word_of(v[0][3], i >> 1), word_of(v[0][2], i >> 1), pick),
                      __builtin_amdgcn_perm(word_of(v[1][1], i >> 1), word_of(v[1][0], i >> 1), pick),
                      __builtin_amdgcn_perm(word_of(v[1][3], i >> 1), word_of(v[1][2], i >> 1), pick));
}

// The workgroup's unit: (request, KV head, split) from the block index.
// MANY: 9 to 16 query heads.
template <int DT, int MODE, bool MANY>
__global__ __launch_bounds__(AT_THR, MODE == AT_SPARSE ? 4 : 3) void attend_kernel(const AttendParams p) {
    __shared__ int2 s_page[AT_CHUNK];           // a page's block, and its tokens | its place in the block << 8
    extern __shared__ float s_dyn[];            // [4 waves][G][AT_PART] for the merge
    __shared__ int s_odd;                       // a wave's sums are not finite
    __shared__ uint32_t s_seen[MODE == AT_WINDOW ? AT_CHUNK : 1];  // a page's places that are seen
    constexpr bool SPARSE = MODE == AT_SPARSE, WINDOW = MODE == AT_WINDOW;
    const int id = blockIdx.x, s = id % p.splits, u = id / p.splits, h = u % p.Hkv, b = u / p.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = MANY ? lane & 15 : lane & 7, quad = lane >> 4;  // the lane's query head
    const int H = p.Hkv * p.G;
    const int L = attend_length(p, b);
    const SeenPages seen = seen_pages(L, WINDOW ? p.window : 0, WINDOW ? p.sinks : 0);
    const int pages = SPARSE ? p.keep << p.bs_shift : seen.pages;
    // Through a window a request's pages are shared out evenly, eight a split at least: a span may be far longer.
    const int pps = WINDOW ? max((pages + p.splits - 1) / p.splits, 8) : p.pps;
    const int k0 = min(s * pps, pages), k1 = min(k0 + pps, pages);
    const int mask = (1 << p.bs_shift) - 1, blocks = (((L + 15) >> 4) + mask) >> p.bs_shift;

    uint4 qf[4];
#pragma unroll
    for (int st = 0; st < 4; ++st)
        qf[st] = col < p.G ? *(const uint4*)(p.q + b * p.q_s0 + (int64_t)(h * p.G + col) * p.q_s1 + 32 * st + 8 * quad)
                           : make_uint4(0, 0, 0, 0);
    const uint16_t* kh = p.kc + (int64_t)h * p.c_s2 + 8 * quad;
    const uint16_t* vh = p.vc + (int64_t)h * p.c_s2 + 8 * (lane & 15);
    if (tid == 0) s_odd = 0;
    for (bool careful = false;; careful = true) {
        float m = -INFINITY, l = 0.f;
        f32x4_t acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        for (int c0 = k0; c0 < k1; c0 += AT_CHUNK) {
            const int count = min(AT_CHUNK, k1 - c0);
            if (c0 != k0) __syncthreads();
            for (int i = tid; i < count; i += AT_THR) {
                const int pg = WINDOW ? seen.page(c0 + i) : c0 + i;
                const int lb = SPARSE ? p.sel[b * p.sel_s0 + h * p.sel_s1 + (pg >> p.bs_shift)] : pg >> p.bs_shift;
                int blk = 0, tokens = 0;
                if (lb >= 0 && lb < blocks) {
                    tokens = min(max(L - 16 * ((lb << p.bs_shift) + (pg & mask)), 0), 16);
                    blk = p.bt[b * p.bt_s0 + lb * p.bt_s1];
                    if (blk < 0 || blk >= p.num_blocks) blk = tokens = 0;  // no block of the cache: no tokens
                }
                s_page[i] = make_int2(blk, tokens | (pg & mask) << 8);
                if constexpr (WINDOW) s_seen[i] = seen.mask(pg);
            }
            __syncthreads();
            for (int i = 2 * wave; i < count; i += 8) {
                int2 e[2];
                int nt[2];
                uint32_t see[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int2 v = s_page[min(i + x, count - 1)];
                    e[x].x = __builtin_amdgcn_readfirstlane(v.x);
                    e[x].y = __builtin_amdgcn_readfirstlane(v.y);
                    nt[x] = i + x < count ? e[x].y & 255 : 0;
                    if constexpr (WINDOW) see[x] = nt[x] ? __builtin_amdgcn_readfirstlane(s_seen[min(i + x, count - 1)]) : 0u;
                }
                float* lg = p.lg + ((int64_t)b * p.Hkv + h) * p.lg_row + (int64_t)(c0 + i) * p.G * 16;  // page i's scores
                if (MODE != AT_SCORES && nt[0] + nt[1] == 0) continue;
                const bool own = col < p.G && (MANY || !(lane & 8));
                uint4 kr[2][4], vr[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    // A page without tokens reads the other one's rows, one with fewer than 16 its last row
                    // again: every address lies in the request's tokens (or, where neither page has a block of the
                    // cache, in block 0), and nothing of them is used.
                    const int2 at = nt[x] ? e[x] : e[x ^ 1];
                    const int last = max(nt[x] ? nt[x] : nt[x ^ 1], 1) - 1;
                    const int64_t base = at.x * p.c_s0 + (int64_t)((at.y >> 8) << 4) * p.c_s1;
#pragma unroll
                    for (int st = 0; st < 4; ++st)
                        kr[x][st] = *(const uint4*)(kh + base + min(lane & 15, last) * p.c_s1 + 32 * st);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        vr[x][j] = *(const uint4*)(vh + base + min(4 * quad + j, last) * p.c_s1);
                }
                float sv[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int st = 0; st < 4; ++st) d = attend_mfma<DT>(kr[x][st], qf[st], d);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sv[x][r] = d[r] * p.sc;
                    if (WINDOW ? see[x] != 0xffffu : nt[x] < 16) {  // tokens past the end or out of sight: no score, and no value that a weight of 0 could turn into NaN
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool ok = WINDOW ? see[x] >> (4 * quad + r) & 1u : 4 * quad + r < nt[x];
                            sv[x][r] = ok ? sv[x][r] : -INFINITY;
                            vr[x][r] = ok ? vr[x][r] : make_uint4(0, 0, 0, 0);
                        }
                    }
                }
                if (MODE == AT_SCORES && own) {
                    *(float4*)(lg + 16 * col + 4 * quad) = make_float4(sv[0][0], sv[0][1], sv[0][2], sv[0][3]);
                    if (i + 1 < count) *(float4*)(lg + 16 * p.G + 16 * col + 4 * quad) = make_float4(sv[1][0], sv[1][1], sv[1][2], sv[1][3]);
                }
                float mx = sv[0][0];
#pragma unroll
                for (int r = 1; r < 8; ++r) mx = fmaxf(mx, sv[r >> 2][r & 3]);
                mx = max_rows(mx);
                if (nt[0] + nt[1] > 0) m = fmaxf(m, AT_LEAST);
                if (__builtin_amdgcn_ballot_w64(mx > m + 15.f) != 0) {
                    const float mn = mx > m + 15.f ? mx - 7.f : m;
                    const float alpha = mn == m ? 1.f : exp2f(m - mn);
                    m = mn;
                    l *= alpha;
#pragma unroll
                    for (int i8 = 0; i8 < 8; ++i8) acc[i8] *= alpha;
                }
                float pe[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool ok = WINDOW ? see[x] >> (4 * quad + r) & 1u : 4 * quad + r < nt[x];
                        pe[x][r] = ok ? exp2f(sv[x][r] - m) * AT_DOWN<DT> : 0.f;
                        l += pe[x][r];
                    }
                if (__builtin_expect(careful, 0)) {
                    const uint4 one = make_uint4(attend_ones<DT>(pe[0][0], pe[0][1]), attend_ones<DT>(pe[0][2], pe[0][3]),
                                                 attend_ones<DT>(pe[1][0], pe[1][1]), attend_ones<DT>(pe[1][2], pe[1][3]));
#pragma unroll
                    for (int i8 = 0; i8 < 8; ++i8) {
                        const uint4 vt = attend_column(vr, i8);
                        acc[i8] = attend_mfma<DT>(make_uint4(vt.x & attend_odd<DT>(vt.x), vt.y & attend_odd<DT>(vt.y),
                                                             vt.z & attend_odd<DT>(vt.z), vt.w & attend_odd<DT>(vt.w)),
                                                  one, acc[i8]);
                    }
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        uint4& v = vr[x >> 2][x & 3];
                        v = make_uint4(v.x & ~attend_odd<DT>(v.x), v.y & ~attend_odd<DT>(v.y), v.z & ~attend_odd<DT>(v.z),
                                       v.w & ~attend_odd<DT>(v.w));
                    }
                }
                // The weights' values, largest first, one a product; up to 8 heads the lanes of the second columns take
                // the second in the first product, the third in the second, the others' second operand being 0.
                uint4 pw[MANY ? 3 : 2];
                if constexpr (!MANY) {
                    const float second = lane & 8 ? 1.f : 0.f;
                    attend_take<DT>(pe[0], second);
                    attend_take<DT>(pe[1], second);
                }
#pragma unroll
                for (int k = 0; k < (MANY ? 3 : 2); ++k) {
                    const uint2 lo = attend_take<DT>(pe[0], 1.f), hi = attend_take<DT>(pe[1], 1.f);
                    pw[k] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
                if (!MANY && !(lane & 8)) pw[1] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int i8 = 0; i8 < 8; ++i8) {
                    const uint4 vt = attend_column(vr, i8);
#pragma unroll
                    for (int k = 0; k < (MANY ? 3 : 2); ++k) acc[i8] = attend_mfma<DT>(vt, pw[k], acc[i8]);
                }
            }
        }
        l = sum_rows(l);
        if constexpr (!MANY) {  // both columns of a head: lanes 8 apart in a row of 16
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[i8][x] += dpp_f<0x128>(acc[i8][x]);  // row_ror:8
        }
        float odd = 0.f;
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8)
#pragma unroll
            for (int x = 0; x < 4; ++x) odd = fmaf(acc[i8][x], 0.f, odd);
        if (col < p.G && odd != 0.f && l == l) s_odd = 1;
        if (col < p.G && (MANY || !(lane & 8))) {
            float* w = s_dyn + (wave * p.G + col) * AT_PART;
            if (quad == 0) {
                w[0] = m;
                w[1] = l;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // dimensions 32 quad + 8 x + i
                *(float4*)(w + 4 + 32 * quad + 8 * x) = make_float4(acc[0][x], acc[1][x], acc[2][x], acc[3][x]);
                *(float4*)(w + 8 + 32 * quad + 8 * x) = make_float4(acc[4][x], acc[5][x], acc[6][x], acc[7][x]);
            }
        }
        __syncthreads();
        if (careful || !s_odd) break;
    }
    for (int i = tid; i < p.G * 128; i += AT_THR) {
        const int g = i >> 7, d = i & 127;
        const float* w = s_dyn + g * AT_PART;
        float M = -INFINITY, lt = 0.f, a = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) M = fmaxf(M, w[k * p.G * AT_PART]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float* r = w + k * p.G * AT_PART;
            // A wave without tokens has reference -inf and sums 0; NaN scores leave sums of NaN, scores of -inf alone 0.
            const float f = r[0] == -INFINITY ? 1.f : exp2f(r[0] - M);
            lt = fmaf(r[1], f, lt);
            a = fmaf(r[4 + d], f, a);
        }
        const int hq = h * p.G + g;
        if (p.splits == 1) store_f(p.out, b * p.o_s0 + hq * p.o_s1 + d, DT, M == -INFINITY ? 0.f : a / lt);
        if (p.splits > 1 || MODE == AT_SCORES) {
            float* pp = p.part + (((int64_t)b * H + hq) * p.splits + s) * AT_PART;
            if (d == 0) *(float4*)pp = make_float4(M, lt, 0.f, 0.f);
            pp[4 + d] = a;
        }
    }
}

// A head's splits joined by one wave: lane s holds the factors of splits s and s + 64, and sums dimensions 2 s
// and 2 s + 1, eight splits' loads in flight.
template <int DT>
__device__ __forceinline__ void attend_merge_head(const AttendParams& p, int b, int hq) {
    static_assert(AT_MAX_SPLITS <= 128, "two splits a lane");
    const int lane = threadIdx.x & 63;
    const float* pp = p.part + ((int64_t)b * p.Hkv * p.G + hq) * p.splits * AT_PART;
    float m[2], f[2], lt = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int s = lane + 64 * x;
        m[x] = s < p.splits ? pp[s * AT_PART] : -INFINITY;
        f[x] = s < p.splits ? pp[s * AT_PART + 1] : 0.f;
    }
    const float M = wave_max(fmaxf(m[0], m[1]));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float l = f[x];
        f[x] = m[x] == -INFINITY ? 1.f : exp2f(m[x] - M);
        lt = fmaf(l, f[x], lt);
    }
    lt = wave_sum(lt);
    float2 a = make_float2(0.f, 0.f);
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
        float2 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = *(const float2*)(pp + min(s0 + u, p.splits - 1) * AT_PART + 4 + 2 * lane);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s0 < 64 ? f[0] : f[1]), (s0 + u) & 63));
            if (s0 + u < p.splits) {
                a.x = fmaf(v[u].x, fs, a.x);
                a.y = fmaf(v[u].y, fs, a.y);
            }
        }
    }
    const int64_t o = b * p.o_s0 + hq * p.o_s1 + 2 * lane;
    store_f(p.out, o, DT, M == -INFINITY ? 0.f : a.x / lt);
    store_f(p.out, o + 1, DT, M == -INFINITY ? 0.f : a.y / lt);
}

// Splits per unit (request and KV head) of at most `pages` pages: workgroups for `per_cu` a CU, `least` pages a
// split at least.
inline int attend_splits(int64_t units, int pages, int per_cu, int least) {
    const int64_t s = std::min<int64_t>((per_cu * (int64_t)device_cus() + units - 1) / units, (pages + least - 1) / least);
    return (int)std::max<int64_t>(1, std::min<int64_t>(s, AT_MAX_SPLITS));
}

inline int block_shift(int block_size) {
    for (int s = 0; s < 16; ++s)
        if (block_size == (16 << s)) return s;
    return -1;
}

// The checks and fields that both decodes share; STARKV_OK or the error's code.
inline int attend_setup(AttendParams& p, const char* what, const void* query, int64_t q_s0, int64_t q_s1,
                        const void* k_cache, const void* v_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype,
                        int block_size, int64_t num_blocks, const int32_t* block_table, int64_t bt_s0, int64_t bt_s1,
                        int bt_width, const int32_t* seq_lens, int n, int num_heads, int num_kv_heads, float scale,
                        void* out, int64_t o_s0, int64_t o_s1, const void* workspace) {
    SKV_CHECK(query && k_cache && v_cache && block_table && seq_lens && out && workspace, "%s: null pointer", what);
    SKV_CHECK(num_kv_heads >= 1 && num_heads >= num_kv_heads && num_heads % num_kv_heads == 0 &&
                  num_heads / num_kv_heads <= AT_MAX_GROUP,
              "%s: %d query heads over %d KV heads (1 to 16 each)", what, num_heads, num_kv_heads);
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "%s: bf16 or fp16", what);
    SKV_CHECK(block_shift(block_size) >= 0, "%s: block_size must be 16 times a power of two", what);
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff && bt_width >= 1, "%s: empty cache or block table", what);
    SKV_CHECK(((uintptr_t)query | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                  (q_s0 | q_s1 | c_s0 | c_s1 | c_s2) % 8 == 0 && (uintptr_t)workspace % 16 == 0,
              "%s: rows must be 16-byte aligned", what);
    p.q = (const uint16_t*)query; p.q_s0 = q_s0; p.q_s1 = q_s1;
    p.kc = (const uint16_t*)k_cache; p.vc = (const uint16_t*)v_cache;
    p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.bs_shift = block_shift(block_size); p.num_blocks = num_blocks;
    p.bt = block_table; p.bt_s0 = bt_s0; p.bt_s1 = bt_s1;
    p.seq_lens = seq_lens;
    p.span = (int)std::min<int64_t>((int64_t)bt_width * block_size, 0x7ffffff0);
    p.n = n; p.Hkv = num_kv_heads; p.G = num_heads / num_kv_heads;
    p.sc = scale * AT_LOG2E;
    p.out = (uint16_t*)out; p.o_s0 = o_s0; p.o_s1 = o_s1;
    return STARKV_OK;
}

template <int MODE>
inline int attend_launch(void* stream, int dtype, const AttendParams& p) {
    SKV_CHECK((int64_t)p.n * p.Hkv * p.splits < 1 << 23, "%d requests of %d KV heads in one call", p.n, p.Hkv);
    const dim3 grid((unsigned)((int64_t)p.n * p.Hkv * p.splits));
    const size_t lds = (size_t)4 * p.G * AT_PART * 4;
    const bool bf = dtype == STARKV_BF16;
    const void* fn = p.G <= 8 ? bf ? (const void*)&attend_kernel<STARKV_BF16, MODE, false>
                                   : (const void*)&attend_kernel<STARKV_F16, MODE, false>
                              : bf ? (const void*)&attend_kernel<STARKV_BF16, MODE, true>
                                   : (const void*)&attend_kernel<STARKV_F16, MODE, true>;
    void* args[] = {(void*)&p};
    SKV_HIP(hipLaunchKernel(fn, grid, dim3(AT_THR), args, lds, (hipStream_t)stream));
    return STARKV_OK;
}

}  // namespace starkv
