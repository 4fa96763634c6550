// The 8-bit cache of an uncompressed layer, [num_blocks, block_size, H_kv, 128] codes of one byte for keys and
// for values, and an exponent of one byte for each block, head and of the two: [num_blocks, H_kv, 2].
//
// A value is code * 2^exponent. Codes are int8 in [-127, 127] or e4m3 up to 448. Scales are powers of two, so
// dividing by one and multiplying by it again is exact, a code's only error is its own rounding (half a step,
// ties to even), and a block whose exponent grows by d has its codes c -> c 2^-d rounded once more: e4m3 codes
// keep all their bits but subnormal ones, int8 codes lose d. A scale of amax / 127 would hold up to one bit more in
// an int8 code (half a bit on average) and would round every value twice, once in its division.
//
// The exponent of values up to a: the least e >= -126 (2^e is a normal number) with a <= 127 2^e, or 448 2^e. A block that
// was given an infinity or NaN has no such exponent: it gets C8_NAN, and its head's values are NaN until the block is
// begun anew (int8 has no code for either, e4m3 none for an infinity).
#pragma once

#include "common.hpp"

namespace starkv {

constexpr int C8_LEAST = -126;
constexpr int C8_NAN = -128;
constexpr int C8_MAX_BLOCK = 1024;  // tokens a block

typedef _Float16 c8_half2 __attribute__((ext_vector_type(2)));
typedef float c8_float2 __attribute__((ext_vector_type(2)));

// The exponent of values whose largest magnitude has these fp32 bits.
template <int CT>
__device__ __forceinline__ int c8_exponent(uint32_t top) {
    const int x = (int)(top >> 23);
    if (x == 255) return C8_NAN;
    // a = m 2^(x - 126), m in [1/2, 1): 127 2^e is 127/128 2^(e + 7), 448 2^e is 7/8 2^(e + 9).
    const uint32_t limit = CT == STARKV_I8 ? 0x7e0000u : 0x600000u;
    return max(x - 126 - (CT == STARKV_I8 ? 7 : 9) + ((top & 0x7fffffu) > limit), C8_LEAST);
}

// 2^e for e in [-126, 127], NaN for C8_NAN.
__device__ __forceinline__ float c8_scale(int e) {
    return e == C8_NAN ? __builtin_nanf("") : __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four values as codes; each at most 127 or 448.
template <int CT>
__device__ __forceinline__ uint32_t c8_pack(float a, float b, float c, float d) {
    if constexpr (CT == STARKV_I8) {
        const uint32_t i = (uint32_t)(int)__builtin_rintf(a) & 255u, j = (uint32_t)(int)__builtin_rintf(b) & 255u;
        const uint32_t k = (uint32_t)(int)__builtin_rintf(c) & 255u, l = (uint32_t)(int)__builtin_rintf(d);
        return i | j << 8 | k << 16 | l << 24;
    } else {
        return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
    }
}

// Four codes as values, before their exponent.
template <int CT>
__device__ __forceinline__ void c8_values(uint32_t w, float (&o)[4]) {
    if constexpr (CT == STARKV_I8) {
        o[0] = (float)(int8_t)w;
        o[1] = (float)(int8_t)(w >> 8);
        o[2] = (float)(int8_t)(w >> 16);
        o[3] = (float)(int8_t)(w >> 24);
    } else {
        const c8_float2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        o[0] = lo[0];
        o[1] = lo[1];
        o[2] = hi[0];
        o[3] = hi[1];
    }
}

// Four codes as fp16, exactly: an operand word pair of a matrix instruction. int8: code + 128 in the low byte of
// 1024 + (code + 128), less 1152.
template <int CT>
__device__ __forceinline__ uint2 c8_halves(uint32_t w) {
    if constexpr (CT == STARKV_I8) {
        const uint32_t u = w ^ 0x80808080u;
        const c8_half2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
        const c8_half2 lo = __builtin_bit_cast(c8_half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
        const c8_half2 hi = __builtin_bit_cast(c8_half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
        return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    } else {
        const c8_half2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
        const c8_half2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
        return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    }
}

// block_size as a shift, -1 where an 8-bit cache cannot have it.
inline int c8_block_shift(int block_size) {
    for (int s = 4; (1 << s) <= C8_MAX_BLOCK; ++s)
        if (block_size == (1 << s)) return s;
    return -1;
}

}  // namespace starkv
