// The 8-bit key/value cache: how a page is laid out, and how a row becomes codes and codes become values.
//
// A page holds 16 tokens. What it keeps of one kv head is one record of 32 head_dim + 32 bytes, contiguous, so that one copy brings all of it:
//   codes of K (16 rows of head_dim bytes), codes of V, the 16 exponents of K, the 16 of V.
// A row of a token (K or V of one kv head) has one exponent e, a byte b = e + 127; a value is code * 2^e. The code is fp8 e4m3, or a
// whole number of 8 bits. e is the smallest exponent with max|x| 2^-e <= 448 (127), not below -100; a row of zeros has e = 0; a row that is not finite, or
// would want an exponent above 100 (a value beyond 448 * 2^100), is NaN: b = 255 and codes 0. Powers of two, because then scaling rounds nothing: a
// value has one rounding (x 2^-e to its code), every stored value is exact in bfloat16, and attention over this cache is attention over the
// bfloat16 cache that holds the same values. (A scale max / 127 would use up to one bit more of the whole numbers; e4m3 has its steps relative to the value and
// gains nothing.)
// Rows lie in pieces of 16 bytes, piece c of key t at number L = t (head_dim / 16) + c, stored at L with some bits turned over (kvq_turn): so the lanes that
// a decode warp reads one plane with fall into different banks, without a copy that swizzles.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

enum { KVQ_E4M3 = 0, KVQ_INT8 = 1 };
constexpr int KVQ_PAGE = 16;
constexpr int KVQ_LEAST = -100, KVQ_MOST = 100, KVQ_NAN = 255;

__host__ __device__ __forceinline__ constexpr int kvq_record(int hd) { return 2 * KVQ_PAGE * hd + 2 * KVQ_PAGE; }
// What a piece's number in its plane is xored with: K of heads of 128 and 256, V of 64, 128 and 256.
__host__ __device__ __forceinline__ constexpr int kvq_turn(int hd, bool v, int key) {
    return v ? (hd == 64 || hd == 128 || hd == 256 ? ((key >> 1) & 3) << 1 : 0) : (hd == 128 || hd == 256 ? (key & 1) << 2 : 0);
}

// The exponent's byte of a row from the bits of its largest magnitude (the largest of the rows' bits without sign, as whole numbers: a NaN is above
// infinity, which is above all others).
template <int KIND>
__device__ __forceinline__ int kvq_exponent(uint32_t most) {
    if (most == 0u) return 127;
    int e = (int)(most >> 23) - 127 - (KIND == KVQ_E4M3 ? 8 : 6);
    e += (most & 0x7fffffu) > (KIND == KVQ_E4M3 ? 0x600000u : 0x7e0000u);       // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    if (e > KVQ_MOST) return KVQ_NAN;             // (a NaN's or an infinity's bits end here too)
    return max(e, KVQ_LEAST) + 127;
}
// 2^-e, what a row is multiplied by before its codes are rounded; 0 for a row that is NaN (its codes are then 0 whatever x is: see kvq_codes4).
__device__ __forceinline__ float kvq_inverse(int b) { return b == KVQ_NAN ? 0.f : __int_as_float((254 - b) << 23); }
// 2^e; NaN for a row that is NaN.
__device__ __forceinline__ float kvq_power(int b) { return __int_as_float(b << 23 | (b + 1 >> 8) << 22); }

// Codes of four values (already times 2^-e), the first in the lowest byte; nearest, ties to even.
template <int KIND>
__device__ __forceinline__ uint32_t kvq_codes4(float a, float b, float c, float d) {
    if (KIND == KVQ_E4M3) {
        uint16_t lo, hi;                          // (the second operand becomes the lower byte)
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    return (uint32_t)(__float2int_rn(a) & 255) | (uint32_t)(__float2int_rn(b) & 255) << 8 | (uint32_t)(__float2int_rn(c) & 255) << 16 |
           (uint32_t)(__float2int_rn(d) & 255) << 24;
}

// Two codes as two halves (exact: e4m3 and whole numbers up to 127 have at most seven bits), the lower code in the lower half. `pair`: two codes for
// e4m3; for whole numbers the two codes with their sign bit turned over, as bytes 0 and 1 (or 2 and 3 with HIGH) of a word.
__device__ __forceinline__ uint32_t kvq_halves_e4m3(uint16_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(pair));
    return h;
}
// 1024 + u as a half is 0x6400 + u for u = 0 .. 255, u = code + 128: one subtraction leaves the code.
template <bool HIGH>
__device__ __forceinline__ uint32_t kvq_halves_int8(uint32_t turned) {
    const uint32_t m = __byte_perm(turned, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    uint32_t h;
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(h) : "r"(m), "r"(0x64806480u));     // 1152
    return h;
}
// The two halves of a word of four codes: bytes 0 and 1, bytes 2 and 3. For whole numbers `w` has its sign bits turned over (kvq_raw).
template <int KIND>
__device__ __forceinline__ uint32_t kvq_raw(uint32_t w) { return KIND == KVQ_E4M3 ? w : w ^ 0x80808080u; }
template <int KIND>
__device__ __forceinline__ uint32_t kvq_low(uint32_t w) { return KIND == KVQ_E4M3 ? kvq_halves_e4m3((uint16_t)(w & 0xffffu)) : kvq_halves_int8<false>(w); }
template <int KIND>
__device__ __forceinline__ uint32_t kvq_high(uint32_t w) { return KIND == KVQ_E4M3 ? kvq_halves_e4m3((uint16_t)(w >> 16)) : kvq_halves_int8<true>(w); }
