// ghip_mx.h -- the codes of a quantized KV cache: blocks of 32 elements, E4M3 (8
// bits) or E2M1 (4 bits, two to a byte, the first in the low bits), each with a
// scale 2^(byte - 127) (E8M0; byte 255: the block is NaN).
//
// gfx950 converts two codes and their scale in one instruction.  A code times a
// power of two has at most 4 significant bits, so bfloat16 holds it exactly (as long as
// it is a normal number: below 2^-126 it may come out as 0), and so does what
// is computed from it as from a bfloat16 cache.
#pragma once
#include "ghip_common.h"

typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 mx_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_h8 __attribute__((ext_vector_type(8)));
typedef float mx_f2 __attribute__((ext_vector_type(2)));
typedef short mx_s2 __attribute__((ext_vector_type(2)));

// the scale that a byte stands for (255: infinity's bits, which the conversions take as NaN)
DEV float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The largest element of a block as bits without a sign (anything from infinity's on:
// the block becomes NaN) -> its scale's byte.  With BITS 8 the least 2^e with max <= 448 2^e
// = 0.875 2^(e + 9); with 4, max <= 7 2^e = 0.875 2^(e + 3): what lies between 6 and 7 becomes
// 6, which costs less than a scale twice as large for the other elements (error of
// normal values 0.112 of their size, 0.115 with 6 or 8 for 7).  e >= -100, where the
// elements of a code's size are still normal numbers of 32 bits.
template <int BITS>
DEV uint32_t mx_scale_of(uint32_t big) {
    const int e = (int)(big >> 23) + 1 - (BITS == 8 ? 9 : 3) + ((big & 0x7fffff) > 0x600000);
    return big >= 0x7f800000 ? 255 : max(e, 27);
}

// Eight elements -> their codes, each rounded to nearest, ties to the even code.
template <int BITS>
struct MxCodes {
    uint32_t w[BITS / 4];
};
template <int BITS>
DEV MxCodes<BITS> mx_encode(const float (&x)[8], uint32_t byte) {
    MxCodes<BITS> c;
    const float s = mx_scale(byte);
#pragma unroll
    for (int i = 0; i < BITS / 4; i++) c.w[i] = 0;
    if (byte == 255) return c;
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mx_s2 w = {0, 0};
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], s, false);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], s, true);
            c.w[i] = __builtin_bit_cast(uint32_t, w);
        }
    } else {
        c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.w[0], x[0], x[1], s, 0);
        c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.w[0], x[2], x[3], s, 1);
        c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.w[0], x[4], x[5], s, 2);
        c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.w[0], x[6], x[7], s, 3);
    }
    return c;
}

// Codes 2 I, 2 I + 1 of a word of them as 32-bit floats; eight codes (2 words, or 1) as
// bfloat16.
template <int BITS, int I>
DEV mx_f2 mx_pair(uint32_t w, float s) {
    if constexpr (BITS == 8) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, I & 1);
    else return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, I);
}
template <int BITS>
DEV mx_bf8 mx_eight(const uint32_t *w, float s, mx_bf8) {
    mx_bf2 p[4];
    if constexpr (BITS == 8) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, false);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, false);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, true);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 3);
    }
    mx_bf8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = p[i / 2][i & 1];
    return r;
}
template <int BITS>
DEV mx_h8 mx_eight(const uint32_t *w, float s, mx_h8) {
    mx_h2 p[4];
    if constexpr (BITS == 8) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], s, false);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], s, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], s, false);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], s, true);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 0);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 1);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 2);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 3);
    }
    mx_h8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = p[i / 2][i & 1];
    return r;
}
template <int BITS>
DEV mx_bf8 mx_eight(const uint32_t *w, float s) { return mx_eight<BITS>(w, s, mx_bf8{}); }

// float16 holds a code times 2^e exactly too, if e is in a range: with 8 bits, all of 2^-9 .. 448, -15 .. 7;
// with 4, all of 0.5 .. 6, -23 .. 13.  A cache's elements are taken 2^HOME times, so that the
// range lies about what they are like: blocks whose largest is 2^-14 .. 224, or 2^-21 .. 57344.
// Exact elements are not all that a sum of products needs, so tiles are computed with as float16 only if
//   keys:   what q's second term leaves off (2^-25 of units in which the row's largest element is 2^14 .. 2^15)
//           moves no score by more than 2^-24, in log2 units: D 2^-25 times the largest code, scale and unit;
//   values: what p's terms leave off (2^-25, of 2^8 or more that a row's largest p is) does not outweigh the
//           rounding of a sum of as many products in 32 bits: the largest elements of all blocks lie within
//           2^9 of one another (codes of STRONG or more, scales at most 2^APART apart).
// And the matrix cores line products up as if an operand below 2^-14 were 2^-14, so a sum whose operands
// are all smaller has fewer bits (measured: values of 2^-23 cost 2^-17 of the output).  So no value that is not 0 lies
// below 2^-17 (2^-38 of p a product: 2^-21 of the element at worst); of keys it is 2^-23 a product, in units of
// 2^-(k + HOME) of a score, of which k + HOME >= SMALL makes too little to count.
// A block of zeros counts as a key of any scale, and as values too weak.
template <int BITS>
struct MxHalf {
    static constexpr int HOME = BITS == 8 ? 8 : 0, SMALL = 4;
    // the bytes of scales, from .. to
    static constexpr int KEYS = 127 - (BITS == 8 ? 15 : 23) - HOME, VALUES = 127 - (BITS == 8 ? 8 : 16) - HOME,
                              TO = 127 + (BITS == 8 ? 7 : 13) - HOME;
    static constexpr int LARGEST = BITS == 8 ? 448 : 6, STRONG = BITS == 8 ? 64 : 2, APART = BITS == 8 ? 6 : 7;
    static_assert((LARGEST << APART) <= STRONG << 9, "values within 2^9 of one another");
    // not 0: one of these BITS / 2 words' codes is STRONG or more
    static __device__ __forceinline__ uint32_t strong(const uint32_t (&x)[BITS / 2]) {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < BITS / 2; i++) r |= BITS == 8 ? (x[i] & 0x7f7f7f7f) + 0x18181818 : x[i];  // (0x68 is 64)
        return r & (BITS == 8 ? 0x80808080 : 0x44444444);
    }
    // ... is not 0
    static __device__ __forceinline__ uint32_t any(const uint32_t (&x)[BITS / 2]) {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < BITS / 2; i++) r |= x[i];
        return r & (BITS == 8 ? 0x7f7f7f7f : 0x77777777);
    }
    // The largest scale of keys for rows of q of which the largest is held 2^k times
    static __device__ __forceinline__ int largest_scale(int k, int D) { return k + HOME < SMALL ? 0 : 128 + k - (32 - __builtin_clz(D * LARGEST - 1)); }
};
