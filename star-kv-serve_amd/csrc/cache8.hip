// The 8-bit cache's write and read back (cache8.hpp has what it holds).
//
// A write puts n tokens' keys and values into their slots. Per block that it touches, head, and of keys and values: e_new
// is the exponent of its own tokens' largest magnitude; where the block's first token is among them the block
// begins anew with it, else the exponent becomes max(e_old, e_new), and where that is more than e_old the codes
// that are there are rounded to it. All tokens of a block have to be known together: one workgroup does a whole
// block, the one of the block's token that leads (its other tokens' workgroups end).
//
// Up to WR_FEW tokens (a decode step) each workgroup finds its block's tokens by looking through all slots, which every
// workgroup reads from L2: one launch. More (prompts) write each token's index to its slot of a map first,
// [num_blocks * block_size] of the workspace, which is not cleared: an entry counts where the slot of the token that
// it names is the entry's own. Measured, one against the other: a step of 512 requests of 8 heads, each in a block of its own,
// 4.1 against 24 us, of 1024 4.9 against 30 (of 32 heads 10 against 31), of 2048 9.7 against 30; a prompt of 512 tokens of 8
// heads 6.6 against 10.7, of 1024 9.6 against 10.9 (of 32 heads 20 against 13), of 2048 12.7 against 11.5 (28 against 16).
// The map's workgroups do up to WR_RUN blocks one after the other, which is what a step of many requests pays there. The host
// does not see which of the two a call is, so the limit is the steps': prompts of 700 to 1024 tokens of 32 heads pay up to 7 us.
//
// A workgroup of the first kind has 4 heads, a wave each, and up to 16 where there would be more than WR_WIDE workgroups: 4 heads
// take a prompt of 64 tokens of 32 heads from 12.6 to 6.1 us, 16 a step of 1024 tokens of 32 heads from 20 to 9.3. In blocks
// of 32 it begins with 2 heads, in larger ones with one, up to WR_WIDE_LARGE workgroups: 300 tokens of 32 heads in blocks of 64 66 ->
// 24 us, a step of 300 7.8 -> 11.
//
// A wave takes a head of the block, keys and values: four rows of 256 bytes a load, largest magnitudes as integer bits
// (NaN is above infinity, which is above all others), rows kept in registers from the first look to the rounding where there
// are at most 16; of more, 2 or 4 waves share a head and meet in LDS (11400 tokens of 32 heads in blocks of 64 191 -> 82 us, of
// 1024 999 -> 163). A block with one token (a step's) is write_single's. Rows are read past the caches: the codes stay there for
// what reads them next (11400 tokens of 32 heads written and read back 130 -> 105 us).
//
// Bound by memory, and for small calls by latency: a step of 64 tokens of 8 heads takes 3.8 us, of which a launch in a graph
// is 2 (4.3 under the profiler); codes that the step has to round again add 2.4. Four prompts of 11407 tokens of 32 heads, 187 MB in and
// 93 out: 56 us, 5.0 TB/s; the copy of 2 GiB runs at 4.9.
#include <algorithm>

#include "cache8.hpp"

namespace starkv {

namespace {

constexpr int WR_THR = 256;
constexpr int WR_FEW = 1024;   // tokens that a workgroup looks through
constexpr int WR_WIDE = 1024;  // workgroups of few tokens: more heads each rather than more, in blocks of 16;
constexpr int WR_WIDE_LARGE = 4096;  // in larger ones
constexpr int WR_RUN = 16;   // tokens of a workgroup of a larger write
constexpr int WR_HELD = 64;  // places of a block that are looked through once

struct Write8Params {
    const uint8_t* src[2]; int64_t s0[2], s1[2];   // keys, values: bytes
    uint8_t* codes[2]; int64_t c_s0, c_s1, c_s2;   // bytes
    int8_t* ex; int64_t x_s0, x_s1;                // [num_blocks][H][2]
    int shift; int64_t num_blocks;                 // block_size = 1 << shift
    const void* slots; int slot64;
    int n, H;
    int32_t* map;                                  // larger writes
};

__device__ __forceinline__ int64_t slot_of(const Write8Params& p, int t) {
    const int64_t s = p.slot64 ? ((const int64_t*)p.slots)[t] : (int64_t)((const int32_t*)p.slots)[t];
    return s >= 0 && s >> p.shift < p.num_blocks ? s : -1;
}

template <int CTL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTL, 0xF, 0xF, true));
}

// The largest of the values of a row of 16 lanes, and of the wave's, in every lane (as row16_max and wave_max).
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
    return dpp_umax<0x140>(dpp_umax<0x141>(dpp_umax<0x4E>(dpp_umax<0xB1>(v))));
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = row_umax(v);
    const auto x = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(x[0], x[1]);
    const auto y = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(y[0], y[1]);
}

// Eight 16-bit values as fp32.
template <int DT>
__device__ __forceinline__ void values8(const uint4& w, float (&f)[8]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == STARKV_BF16) {
            f[2 * k] = __uint_as_float(ws[k] << 16);
            f[2 * k + 1] = __uint_as_float(ws[k] & 0xffff0000u);
        } else {
            f[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(ws[k] & 0xffffu));
            f[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(ws[k] >> 16));
        }
    }
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The larger of two pairs of 16-bit magnitudes: their order is that of their bits, for either type.
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

__device__ __forceinline__ uint32_t pair_max(uint32_t top, const uint4& w) {
    constexpr uint32_t M = 0x7fff7fffu;
    return pair_max(top, pair_max(pair_max(w.x & M, w.y & M), pair_max(w.z & M, w.w & M)));
}

// The fp32 bits of the larger of a pair of magnitudes.
template <int DT>
__device__ __forceinline__ uint32_t top_bits(uint32_t pair) {
    const uint32_t x = max(pair & 0xffffu, pair >> 16);
    if constexpr (DT == STARKV_BF16) return x << 16;
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)x));
}

template <int CT, int DT>
__device__ __forceinline__ uint2 encode(const uint4& w, float inv) {
    float f[8];
    values8<DT>(w, f);
    return make_uint2(c8_pack<CT>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                      c8_pack<CT>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

// The exponent of a block's head after a write whose own is e.
__device__ __forceinline__ int joined(int old, int e, bool fresh) {
    return fresh ? e : old == C8_NAN || e == C8_NAN ? C8_NAN : max(old, e);
}

// The codes of places first, first + step, ... that have no token now (tok < 0) to an exponent that is `by` more, eight of a
// place to a lane: the loads of DEEP places go out before the first is rounded.
template <int CT, int DEEP, class Tok>
__device__ __forceinline__ void lessen(uint8_t* dst, int64_t stride, int first, int step, int size, Tok tok, int by) {
    const float less = c8_scale(-min(by, 126));
    for (int at = first; at < size; at += DEEP * step) {
        uint2 w[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (at + step * i < size) w[i] = *(const uint2*)(dst + (at + step * i) * stride);
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            if (at + step * i >= size || tok(at + step * i) >= 0) continue;
            float a[4], b[4];
            c8_values<CT>(w[i].x, a);
            c8_values<CT>(w[i].y, b);
            *(uint2*)(dst + (at + step * i) * stride) =
                make_uint2(c8_pack<CT>(a[0] * less, a[1] * less, a[2] * less, a[3] * less),
                           c8_pack<CT>(b[0] * less, b[1] * less, b[2] * less, b[3] * less));
        }
    }
}

// Rows of 4 KEEP of a block's tokens, keys and values, of one head: a wave's lanes have 16 bytes of 4 rows each.
constexpr int KEEP = 4;
struct Rows8 {
    uint4 w[2][KEEP];
    int old[2];  // the exponents that are there
};

__device__ __forceinline__ void load_head(const Write8Params& p, Rows8& r, int blk, int h, const int* tok, const uint16_t* list,
                                          int count) {
    const int lane = threadIdx.x & 63, row = lane >> 4, d = lane & 15;
    const int8_t* ex = p.ex + blk * p.x_s0 + h * p.x_s1;
#pragma unroll
    for (int z = 0; z < 2; ++z) r.old[z] = ex[z];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int at = 4 * i + row;
        const int64_t t = at < count ? tok[list[at]] : -1;
#pragma unroll
        for (int z = 0; z < 2; ++z)
            r.w[z][i] = t >= 0 ? load_once16(p.src[z] + h * p.s1[z] + 16 * d + t * p.s0[z]) : make_uint4(0, 0, 0, 0);
    }
}

// One block's head by one wave, keys and values. tok[place]: the token of each place or -1; list: the places that have
// one, `count` of them; r: the first rows of them.
template <int CT, int DT, int DEEP>
__device__ __forceinline__ void write_head(const Write8Params& p, const Rows8& r, int blk, int h, const int* tok,
                                           const uint16_t* list, int count) {
    const int lane = threadIdx.x & 63, row = lane >> 4, d = lane & 15;
    int8_t* ex = p.ex + blk * p.x_s0 + h * p.x_s1;
    const bool fresh = tok[0] >= 0;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        uint8_t* dst = p.codes[z] + blk * p.c_s0 + h * p.c_s2 + 8 * d;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) top = pair_max(top, r.w[z][i]);
        const int old = r.old[z], e = joined(old, c8_exponent<CT>(wave_umax(top_bits<DT>(top))), fresh);
        if (!fresh && e != old && e != C8_NAN)  // the codes that are there, to the new exponent
            lessen<CT, DEEP>(dst, p.c_s1, row, 4, 1 << p.shift, [&](int at) { return tok[at]; }, e - old);
        const float inv = e == C8_NAN ? 0.f : c8_scale(-e);
        const auto put = [&](int at, const uint4& w) {
            *(uint2*)(dst + list[at] * p.c_s1) = e == C8_NAN ? make_uint2(0, 0) : encode<CT, DT>(w, inv);
        };
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (4 * i + row < count) put(4 * i + row, r.w[z][i]);
        if (lane == 0 && e != old) ex[z] = (int8_t)e;
    }
}

struct Block8Shared {
    int tok[C8_MAX_BLOCK];        // the token of each place, -1
    uint16_t list[C8_MAX_BLOCK];  // the places that have one
    int count, lead;
    uint32_t top[2][2][WR_THR / 64];  // by turn, keys or values, wave
};

// The places with tokens, from tok; the workgroup's threads meet on both sides.
__device__ __forceinline__ void list_places(Block8Shared& sh, int shift) {
    __syncthreads();
    for (int i = threadIdx.x; i < 1 << shift; i += WR_THR)
        if (sh.tok[i] >= 0) sh.list[atomicAdd(&sh.count, 1)] = (uint16_t)i;
    __syncthreads();
}

// Up to four heads of a block with one token by a wave: a step writes one token of a block. 16 lanes take the token's row of
// a head, so that the heads' latencies pass together; codes that have to be rounded again are the whole wave's, four places
// at a time, one head after the other.
template <int CT, int DT, int DEEP>
__device__ __forceinline__ void write_single(const Write8Params& p, int blk, int h0, int h1, int t, int place) {
    const int lane = threadIdx.x & 63, row = lane >> 4, d = lane & 15, h = h0 + WR_THR / 64 * row;
    const bool on = h < h1;
    int8_t* ex = p.ex + blk * p.x_s0 + h * p.x_s1;
    uint4 w[2] = {};
    int old[2] = {};
    if (on) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            w[z] = load_once16(p.src[z] + h * p.s1[z] + 16 * d + (int64_t)t * p.s0[z]);
            old[z] = ex[z];
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        uint8_t* dst = p.codes[z] + blk * p.c_s0 + 8 * d;
        const int e = joined(old[z], c8_exponent<CT>(row_umax(top_bits<DT>(pair_max(0, w[z])))), place == 0);
        for (uint64_t grown = __ballot(on && d == 0 && place != 0 && e != old[z] && e != C8_NAN); grown; grown &= grown - 1) {
            const int g = __builtin_ctzll(grown), by = __builtin_amdgcn_readlane(e - old[z], g);
            lessen<CT, DEEP>(dst + (h0 + WR_THR / 64 * (g >> 4)) * p.c_s2, p.c_s1, row, 4, 1 << p.shift,
                                [&](int at) { return at == place ? t : -1; }, by);
        }
        if (!on) continue;
        *(uint2*)(dst + h * p.c_s2 + place * p.c_s1) = e == C8_NAN ? make_uint2(0, 0) : encode<CT, DT>(w[z], c8_scale(-e));
        if (d == 0 && e != old[z]) ex[z] = (int8_t)e;
    }
}

// Heads of a block of more than 4 KEEP tokens by teams of 2 or 4 waves (`team` of them), 4 KEEP rows a wave at a time: the first
// ones stay in registers from the first look to the rounding, others are read twice. The largest magnitudes meet in LDS, one
// barrier a head.
template <int CT, int DT, int DEEP>
__device__ __forceinline__ void write_together(const Write8Params& p, Block8Shared& sh, int blk, int h0, int h1, int team) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane >> 4, d = lane & 15;
    const int member = wave & (team - 1), teams = WR_THR / 64 / team, count = sh.count, stride = 4 * KEEP * team;
    const bool fresh = sh.tok[0] >= 0;
    for (int i = 0; h0 + i * teams < h1; ++i) {
        const int h = h0 + i * teams + wave / team;
        const bool on = h < h1;
        int8_t* ex = p.ex + blk * p.x_s0 + h * p.x_s1;
        uint4 w[2][KEEP];
        int old[2] = {0, 0};
        // Rows of places first + 4 i + row of the list.
        const auto load = [&](int z, int first) {
#pragma unroll
            for (int k = 0; k < KEEP; ++k) {
                const int at = first + 4 * k + row;
                w[z][k] = on && at < count ? load_once16(p.src[z] + h * p.s1[z] + 16 * d + (int64_t)sh.tok[sh.list[at]] * p.s0[z])
                                           : make_uint4(0, 0, 0, 0);
            }
        };
        const int own = 4 * KEEP * member;
        uint32_t top[2] = {0, 0};
        for (int first = own + (count - 1 - own) / stride * stride; first >= own; first -= stride) {  // its first rows last
#pragma unroll
            for (int z = 0; z < 2; ++z) load(z, first);
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int k = 0; k < KEEP; ++k) top[z] = pair_max(top[z], w[z][k]);
        }
        if (on) {
#pragma unroll
            for (int z = 0; z < 2; ++z) old[z] = ex[z];
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const uint32_t t = wave_umax(top_bits<DT>(top[z]));
            if (lane == 0) sh.top[i & 1][z][wave] = t;
        }
        __syncthreads();
        if (!on) continue;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            uint32_t t = 0;
            for (int k = 0; k < team; ++k) t = max(t, sh.top[i & 1][z][wave - member + k]);
            uint8_t* dst = p.codes[z] + blk * p.c_s0 + h * p.c_s2 + 8 * d;
            const int e = joined(old[z], c8_exponent<CT>(t), fresh);
            if (!fresh && e != old[z] && e != C8_NAN)
                lessen<CT, DEEP>(dst, p.c_s1, 4 * member + row, 4 * team, 1 << p.shift, [&](int at) { return sh.tok[at]; }, e - old[z]);
            const float inv = e == C8_NAN ? 0.f : c8_scale(-e);
            for (int first = own; first < count; first += stride) {
                if (first > own) load(z, first);
#pragma unroll
                for (int k = 0; k < KEEP; ++k) {
                    const int at = first + 4 * k + row;
                    if (at < count) *(uint2*)(dst + sh.list[at] * p.c_s1) = e == C8_NAN ? make_uint2(0, 0) : encode<CT, DT>(w[z][k], inv);
                }
            }
            if (member == 0 && lane == 0 && e != old[z]) ex[z] = (int8_t)e;
        }
    }
}

// Heads [h0, h1) of a block by a workgroup.
template <int CT, int DT, int DEEP, bool LARGE>
__device__ __forceinline__ void write_heads(const Write8Params& p, Block8Shared& sh, int blk, int h0, int h1) {
    const int wave = threadIdx.x >> 6;
    if (sh.count == 1) {
        const int place = sh.list[0];
        for (int h = h0 + wave; h < h1; h += WR_THR / 16) write_single<CT, DT, DEEP>(p, blk, h, h1, sh.tok[place], place);
        return;
    }
    if (LARGE && sh.count > 4 * KEEP) {
        write_together<CT, DT, DEEP>(p, sh, blk, h0, h1, sh.count > 8 * KEEP ? 4 : 2);
        return;
    }
    for (int h = h0 + wave; h < h1; h += WR_THR / 64) {
        Rows8 r;
        load_head(p, r, blk, h, sh.tok, sh.list, sh.count);
        write_head<CT, DT, DEEP>(p, r, blk, h, sh.tok, sh.list, sh.count);
    }
}

// A workgroup a token and `heads` heads: the block's tokens by looking through all slots.
template <int CT, int DT>
__global__ __launch_bounds__(WR_THR) void write8_few_kernel(const Write8Params p, int heads) {
    __shared__ Block8Shared sh;
    // Consecutive workgroups run on different dies, and of a prompt in order one token of 16 2^s leads its block: within each
    // 8 tokens the order turns by one from block to block, whatever s, else one die would do all of the work.
    const int b = blockIdx.x, tid = threadIdx.x;
    const int t = (b & ~7) | ((b + (b >> 4) + (b >> 7) + (b >> 10)) & 7);
    if (t >= p.n) return;
    const int64_t slot = slot_of(p, t);
    if (slot < 0) return;
    const int blk = (int)(slot >> p.shift), size = 1 << p.shift;
    if (t > 0) {  // behind another of its block: that or one before it leads
        const int64_t before = slot_of(p, t - 1);
        if (before >= 0 && before >> p.shift == blk) return;
    }
    for (int i = tid; i < size; i += WR_THR) sh.tok[i] = -1;
    if (tid == 0) {
        sh.count = 0;
        sh.lead = p.n;
    }
    __syncthreads();
    for (int i = tid; i < p.n; i += WR_THR) {
        const int64_t s = slot_of(p, i);
        if (s >= 0 && s >> p.shift == blk) {
            atomicMax(&sh.tok[s & (size - 1)], i);  // of two tokens with one slot the later
            atomicMin(&sh.lead, i);
        }
    }
    list_places(sh, p.shift);
    if (sh.lead != t) return;
    write_heads<CT, DT, 4, true>(p, sh, blk, blockIdx.y * heads, min((int)(blockIdx.y + 1) * heads, p.H));
}

__global__ __launch_bounds__(WR_THR) void write8_map_kernel(const Write8Params p) {
    const int t = blockIdx.x * WR_THR + threadIdx.x;
    if (t >= p.n) return;
    const int64_t slot = slot_of(p, t);
    if (slot >= 0) p.map[slot] = t;
}

// The token of a slot by the map, -1 where it has none.
__device__ __forceinline__ int mapped(const Write8Params& p, int64_t slot) {
    const int t = p.map[slot];
    return (uint32_t)t < (uint32_t)p.n && slot_of(p, t) == slot ? t : -1;
}

// Whether token t has a slot and the one before it has no lower place of the same block.
__device__ __forceinline__ bool may_lead(const Write8Params& p, int t) {
    const int64_t slot = t < p.n ? slot_of(p, t) : -1, before = t > 0 && t < p.n ? slot_of(p, t - 1) : -1;
    return slot >= 0 && !(before < slot && before >= (slot >> p.shift << p.shift));
}

// A workgroup `runs` times WR_RUN tokens (WR_THR at most) and `heads` heads: the blocks that one of the tokens leads (has the
// lowest place of). 16 threads a token that may lead look through its block's places; what they find of the first
// WR_HELD places stays with them for the block's turn. LARGE: blocks of more than 16 tokens (one run of blocks of 16 with the
// others' registers would leave room for a quarter fewer waves).
template <int CT, int DT, bool LARGE>
__global__ __launch_bounds__(WR_THR) void write8_kernel(const Write8Params p, int runs, int heads) {
    __shared__ Block8Shared sh;
    __shared__ int s_follows[WR_RUN], s_blk[WR_RUN], s_any[WR_THR / WR_RUN];
    const int groups = (p.H + heads - 1) / heads, first_t = blockIdx.x / groups * runs * WR_RUN, group = blockIdx.x % groups;
    const int tid = threadIdx.x, size = 1 << p.shift, mine = tid / WR_RUN, sub = tid % WR_RUN;
    if (!LARGE) runs = 1;
    if (runs > 1) {  // of several runs most have none that may lead
        const uint64_t may = __ballot(tid < runs * WR_RUN && may_lead(p, first_t + tid));
        if (sub == 0) s_any[mine] = (may >> (tid & 48) & 0xffff) != 0;
    }
    for (int r = 0; r < runs; ++r) {
        if (runs > 1) {
            __syncthreads();
            if (!s_any[r]) continue;
        }
        int held[WR_HELD / WR_RUN];
        {
            const int t = first_t + r * WR_RUN + mine;
            const int64_t slot = t < p.n ? slot_of(p, t) : -1, first = slot & ~(int64_t)(size - 1);
            bool follows = LARGE ? !may_lead(p, t) : slot < 0;  // of 16 places the look costs less than the question
            if (sub == 0) {
                s_follows[mine] = follows;
                s_blk[mine] = (int)(slot >> p.shift);
            }
            __syncthreads();
            if (!follows) {
#pragma unroll
                for (int i = 0; i < WR_HELD / WR_RUN; ++i) held[i] = sub + WR_RUN * i < size ? mapped(p, first + sub + WR_RUN * i) : -1;
                follows = p.map[slot] != t;  // another token has the slot too, and the map names that
#pragma unroll
                for (int i = 0; i < WR_HELD / WR_RUN; ++i) follows = follows || (held[i] >= 0 && first + sub + WR_RUN * i < slot);
                // In larger blocks the nearest lower places first: a prompt's token has its neighbour there.
                if (size > WR_HELD)
                    for (int64_t s = slot - 1 - sub; s >= first + WR_HELD; s -= WR_RUN) {
                        follows = follows || mapped(p, s) >= 0;
                        if (__ballot(follows) >> (tid & 48) & 0xffff) break;
                    }
                if (follows) s_follows[mine] = 1;
            }
            __syncthreads();
        }
        for (int j = 0; j < WR_RUN; ++j) {
            if (s_follows[j]) continue;
            const int blk = s_blk[j];
            if (tid == 0) sh.count = 0;
            if (mine == j) {
#pragma unroll
                for (int i = 0; i < WR_HELD / WR_RUN; ++i)
                    if (sub + WR_RUN * i < size) sh.tok[sub + WR_RUN * i] = held[i];
            }
            for (int i = tid + WR_HELD; i < size; i += WR_THR) sh.tok[i] = mapped(p, ((int64_t)blk << p.shift) + i);
            list_places(sh, p.shift);
            write_heads<CT, DT, 1, LARGE>(p, sh, blk, group * heads, min((group + 1) * heads, p.H));
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------
// Rows back: code * 2^exponent, rounded once to 16 or 32 bits
// ---------------------------------------------------------------------------
struct Read8Params {
    const uint8_t* codes[2]; int64_t c_s0, c_s1, c_s2;  // bytes
    const int8_t* ex; int64_t x_s0, x_s1;
    int shift; int64_t num_blocks;
    const void* slots; int slot64;
    int n, H;
    void* out[2];                                       // [n][H][128]
};

// 16 lanes a row of 8 dimensions each, RD_U rows (of keys and of values) a lane, whose slots and then codes are on their way
// together; rows as the results lie, a token's heads side by side. The bound is HBM: 128 bytes read and 256 written a
// row.
constexpr int RD_U = 2;
// Results of 16 bits of more than this many bytes go past the caches (256 MB in the last level), which they would not fit: 11400
// tokens of 32 heads behind their write 105 -> 96 us, 60515 of 8 heads (248 MB) 72 -> 66. Fewer stay there for their reader
// (4096 tokens of 32 heads, 67 MB: 16.8 us, 16.5 past them).
constexpr int64_t RD_ONCE = 128 << 20;

template <bool ONCE>
__device__ __forceinline__ void store_row(uint16_t* to, const uint32_t (&v)[4]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 w = {v[0], v[1], v[2], v[3]};
    if constexpr (ONCE)
        __builtin_nontemporal_store(w, (u32x4*)to);
    else
        *(u32x4*)to = w;
}

template <int CT, int ODT, bool ONCE>
__global__ __launch_bounds__(256) void read8_kernel(const Read8Params p) {
    const uint32_t rows = (uint32_t)p.n * p.H, row0 = blockIdx.x * (16 * RD_U) + (threadIdx.x >> 4);
    const int d = 8 * (threadIdx.x & 15);
    int64_t slot[RD_U];
    uint32_t h[RD_U];
#pragma unroll
    for (int u = 0; u < RD_U; ++u) {
        const uint32_t row = min(row0 + 16 * u, rows - 1), t = row / (uint32_t)p.H;
        h[u] = row - t * p.H;
        slot[u] = p.slot64 ? ((const int64_t*)p.slots)[t] : (int64_t)((const int32_t*)p.slots)[t];
    }
    uint2 w[RD_U][2];
    int e[RD_U][2];
#pragma unroll
    for (int u = 0; u < RD_U; ++u) {
        if (slot[u] < 0 || slot[u] >> p.shift >= p.num_blocks) slot[u] = -1;
        const int64_t s = max(slot[u], (int64_t)0), blk = s >> p.shift;
        const int64_t at = blk * p.c_s0 + (s & ((1 << p.shift) - 1)) * p.c_s1 + h[u] * p.c_s2 + d;
        const int8_t* ex = p.ex + blk * p.x_s0 + h[u] * p.x_s1;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            w[u][z] = *(const uint2*)(p.codes[z] + at);
            e[u][z] = ex[z];
        }
    }
#pragma unroll
    for (int u = 0; u < RD_U; ++u) {
        if (row0 + 16 * u >= rows) break;
        const int64_t to = (int64_t)(row0 + 16 * u) * 128 + d;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const float scale = c8_scale(e[u][z]);
            float a[4], b[4];
            c8_values<CT>(w[u][z].x, a);
            c8_values<CT>(w[u][z].y, b);
            float f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[i] = slot[u] < 0 ? 0.f : a[i] * scale;
                f[4 + i] = slot[u] < 0 ? 0.f : b[i] * scale;
            }
            if constexpr (ODT == STARKV_F32) {
                float4* o = (float4*)((float*)p.out[z] + to);
                o[0] = make_float4(f[0], f[1], f[2], f[3]);
                o[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint16_t lo = ODT == STARKV_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)f[2 * i]) : __builtin_bit_cast(uint16_t, (_Float16)f[2 * i]);
                    const uint16_t hi = ODT == STARKV_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)f[2 * i + 1]) : __builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]);
                    v[i] = (uint32_t)lo | (uint32_t)hi << 16;
                }
                store_row<ONCE>((uint16_t*)p.out[z] + to, v);
            }
        }
    }
}

template <int CT, bool LARGE>
const void* write_pick(bool bf) {
    return bf ? (const void*)&write8_kernel<CT, STARKV_BF16, LARGE> : (const void*)&write8_kernel<CT, STARKV_F16, LARGE>;
}

template <int CT>
const void* read_pick(int dt, bool once) {
    if (dt == STARKV_F32) return (const void*)&read8_kernel<CT, STARKV_F32, false>;
    if (dt == STARKV_F16) return once ? (const void*)&read8_kernel<CT, STARKV_F16, true> : (const void*)&read8_kernel<CT, STARKV_F16, false>;
    return once ? (const void*)&read8_kernel<CT, STARKV_BF16, true> : (const void*)&read8_kernel<CT, STARKV_BF16, false>;
}

}  // namespace

}  // namespace starkv

using namespace starkv;

extern "C" {

size_t starkv_write_kv8_workspace_bytes(int n, int64_t num_blocks, int block_size) {
    if (n <= WR_FEW || num_blocks < 1 || block_size < 1) return 0;
    return (size_t)num_blocks * block_size * 4;
}

int starkv_write_kv8(void* stream, const void* key, int64_t k_s0, int64_t k_s1, const void* value, int64_t v_s0,
                     int64_t v_s1, int dtype, void* k_codes, void* v_codes, int64_t c_s0, int64_t c_s1, int64_t c_s2,
                     int code_type, int8_t* exponents, int64_t x_s0, int64_t x_s1, int block_size, int64_t num_blocks,
                     const void* slot_mapping, int slot_bits, int n, int num_kv_heads, void* workspace,
                     size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && num_kv_heads >= 1 && num_kv_heads <= 65535, "write_kv8: n=%d num_kv_heads=%d (up to 65535)", n, num_kv_heads);
    if (n == 0) return STARKV_OK;
    SKV_CHECK(key && value && k_codes && v_codes && exponents && slot_mapping, "write_kv8: null pointer");
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "write_kv8: keys and values must be bf16 or fp16");
    SKV_CHECK(code_type == STARKV_I8 || code_type == STARKV_E4M3, "write_kv8: codes must be int8 or e4m3");
    SKV_CHECK(slot_bits == 32 || slot_bits == 64, "write_kv8: slot_mapping must be int32 or int64");
    SKV_CHECK(c8_block_shift(block_size) >= 0, "write_kv8: block_size must be 16 times a power of two, at most %d", C8_MAX_BLOCK);
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff, "write_kv8: empty cache");
    SKV_CHECK(((uintptr_t)key | (uintptr_t)value) % 16 == 0 && (k_s0 | k_s1 | v_s0 | v_s1) % 8 == 0 &&
                  ((uintptr_t)k_codes | (uintptr_t)v_codes) % 16 == 0 && (c_s0 | c_s1 | c_s2) % 16 == 0,
              "write_kv8: rows must be 16-byte aligned");
    const size_t need = starkv_write_kv8_workspace_bytes(n, num_blocks, block_size);
    SKV_CHECK(workspace_bytes >= need && (workspace || need == 0) && (uintptr_t)workspace % 16 == 0, "write_kv8: workspace %zu bytes < %zu", workspace_bytes, need);
    Write8Params p;
    p.src[0] = (const uint8_t*)key; p.s0[0] = 2 * k_s0; p.s1[0] = 2 * k_s1;
    p.src[1] = (const uint8_t*)value; p.s0[1] = 2 * v_s0; p.s1[1] = 2 * v_s1;
    p.codes[0] = (uint8_t*)k_codes; p.codes[1] = (uint8_t*)v_codes;
    p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.ex = exponents; p.x_s0 = x_s0; p.x_s1 = x_s1;
    p.shift = c8_block_shift(block_size); p.num_blocks = num_blocks;
    p.slots = slot_mapping; p.slot64 = slot_bits == 64;
    p.n = n; p.H = num_kv_heads;
    p.map = (int32_t*)workspace;
    const bool i8 = code_type == STARKV_I8, bf = dtype == STARKV_BF16;
    if (n <= WR_FEW) {
        const void* fn = i8 ? bf ? (const void*)&write8_few_kernel<STARKV_I8, STARKV_BF16> : (const void*)&write8_few_kernel<STARKV_I8, STARKV_F16>
                            : bf ? (const void*)&write8_few_kernel<STARKV_E4M3, STARKV_BF16> : (const void*)&write8_few_kernel<STARKV_E4M3, STARKV_F16>;
        int heads = 4 >> std::min(p.shift - 4, 2);
        while (heads < 16 && (int64_t)n * ((num_kv_heads + heads - 1) / heads) > (p.shift > 4 ? WR_WIDE_LARGE : WR_WIDE)) heads *= 2;
        void* args[] = {(void*)&p, (void*)&heads};
        SKV_HIP(hipLaunchKernel(fn, dim3((n + 7) / 8 * 8, (num_kv_heads + heads - 1) / heads), dim3(WR_THR), args, 0, (hipStream_t)stream));
        return STARKV_OK;
    }
    hipLaunchKernelGGL(write8_map_kernel, dim3((n + WR_THR - 1) / WR_THR), dim3(WR_THR), 0, (hipStream_t)stream, p);
    SKV_HIP(hipGetLastError());
    const void* fn = p.shift > 4 ? i8 ? write_pick<STARKV_I8, true>(bf) : write_pick<STARKV_E4M3, true>(bf)
                                 : i8 ? write_pick<STARKV_I8, false>(bf) : write_pick<STARKV_E4M3, false>(bf);
    // Of blocks of 16 two heads a wave: the search for a block's tokens is made once for them. Of larger ones as many rows. More
    // tokens than a step has requests are prompts', of which a block's first token leads: up to a block's tokens to a workgroup
    // then, while there are 512 workgroups (in blocks of 64, where one workgroup of four finds something to do: 4 prompts of 2900
    // tokens of 32 heads 144 -> 82 us, 17 of 255 of 8 heads 34 -> 21 with two runs, 29 with four).
    int heads = std::max(8 >> (p.shift - 4), 1), runs = 1;
    const int64_t groups = (num_kv_heads + heads - 1) / heads;
    const auto grid_of = [&](int r) { return ((int64_t)n + r * WR_RUN - 1) / (r * WR_RUN) * groups; };
    if (n > 2 * WR_FEW)
        while (runs < 1 << (p.shift - 4) && runs < WR_THR / WR_RUN && grid_of(2 * runs) >= 512) runs *= 2;
    void* args[] = {(void*)&p, (void*)&runs, (void*)&heads};
    const int64_t grid = grid_of(runs);
    SKV_CHECK(grid < 1ll << 31, "write_kv8: %d tokens of %d heads in one call", n, num_kv_heads);
    SKV_HIP(hipLaunchKernel(fn, dim3((unsigned)grid), dim3(WR_THR), args, 0,
                            (hipStream_t)stream));
    return STARKV_OK;
}

int starkv_read_kv8(void* stream, const void* k_codes, const void* v_codes, int64_t c_s0, int64_t c_s1, int64_t c_s2,
                    int code_type, const int8_t* exponents, int64_t x_s0, int64_t x_s1, int block_size,
                    int64_t num_blocks, const void* slot_mapping, int slot_bits, int n, int num_kv_heads, void* key_out,
                    void* value_out, int out_dtype) {
    clear_error();
    SKV_CHECK(n >= 0 && num_kv_heads >= 1 && num_kv_heads <= 65535, "read_kv8: n=%d num_kv_heads=%d (up to 65535)", n, num_kv_heads);
    if (n == 0) return STARKV_OK;
    SKV_CHECK(k_codes && v_codes && exponents && slot_mapping && key_out && value_out, "read_kv8: null pointer");
    SKV_CHECK(out_dtype >= STARKV_F32 && out_dtype <= STARKV_BF16, "read_kv8: rows of bf16, fp16 or fp32");
    SKV_CHECK(code_type == STARKV_I8 || code_type == STARKV_E4M3, "read_kv8: codes must be int8 or e4m3");
    SKV_CHECK(slot_bits == 32 || slot_bits == 64, "read_kv8: slot_mapping must be int32 or int64");
    SKV_CHECK(c8_block_shift(block_size) >= 0, "read_kv8: block_size must be 16 times a power of two, at most %d", C8_MAX_BLOCK);
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff, "read_kv8: empty cache");
    SKV_CHECK(((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)key_out | (uintptr_t)value_out) % 16 == 0 &&
                  (c_s0 | c_s1 | c_s2) % 16 == 0,
              "read_kv8: rows must be 16-byte aligned");
    Read8Params p;
    p.codes[0] = (const uint8_t*)k_codes; p.codes[1] = (const uint8_t*)v_codes;
    p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.ex = exponents; p.x_s0 = x_s0; p.x_s1 = x_s1;
    p.shift = c8_block_shift(block_size); p.num_blocks = num_blocks;
    p.slots = slot_mapping; p.slot64 = slot_bits == 64;
    p.n = n; p.H = num_kv_heads;
    const bool once = (int64_t)n * num_kv_heads * 512 > RD_ONCE;
    p.out[0] = key_out; p.out[1] = value_out;
    const void* fn = code_type == STARKV_I8 ? read_pick<STARKV_I8>(out_dtype, once) : read_pick<STARKV_E4M3>(out_dtype, once);
    void* args[] = {(void*)&p};
    const int64_t rows = (int64_t)n * num_kv_heads, per = 16 * RD_U;
    SKV_CHECK(rows < 1ll << 31, "read_kv8: %d tokens of %d heads in one call", n, num_kv_heads);
    SKV_HIP(hipLaunchKernel(fn, dim3((unsigned)((rows + per - 1) / per)), dim3(256), args, 0, (hipStream_t)stream));
    return STARKV_OK;
}

}  // extern "C"
