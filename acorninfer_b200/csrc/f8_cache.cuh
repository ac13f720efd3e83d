// The 8-bit key/value cache: what its kernels share.
//
// A row of the cache (the key or the value of one token and kv head, d entries) is held as e4m3 codes and one power of
// two, row = code * 2^e: e is the smallest integer in -120 .. 120 for which 448 * 2^e is not below the row's largest
// magnitude, a code is the nearest e4m3 number (ties to even).  448 = 1.75 * 2^8 is the largest e4m3 number.  Powers of two
// because the products are then exact wherever they are formed: a code has four significant bits, so code * 2^e is a bfloat16
// number (down to 2^-9 * 2^-120, which is a subnormal one), and the attention rounds nothing on the format's behalf.  A row of
// its own for every token and head because such a row is complete when its token is written: nothing is calibrated, and no
// later token changes it.  A row with an infinity or a NaN among its entries holds zeros and the exponent byte 255: the
// queries that read it get NaN, the others do not notice.
//
// Codes: [pages, kv heads, page, d], key and value pages apart.  Exponents: [pages, kv heads, page, 2] bytes, those of a
// token's key and value side by side (e8m0: 2^(byte - 127)), so that the exponents of a (page, head) tile are one run of
// 2 * page bytes, which a bulk copy takes from pages of 8 tokens on.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "attention_mask.cuh"

#define F8_MAX_EXP 120
#define F8_NAN_BYTE 255

// The exponent of a row whose largest magnitude is `most` (finite, >= 0): 2^(e + 8) * 1.75 >= most, from the bits of
// the number (a subnormal one has biased exponent 0 and ends at the lower limit like zero).
__device__ __forceinline__ int f8_row_exponent(float most) {
    const uint32_t b = __float_as_uint(most);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(-F8_MAX_EXP, min(F8_MAX_EXP, e));
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float f8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The number an exponent byte stands for: NaN for 255, 2^-127 (a subnormal number) for 0.
__device__ __forceinline__ float f8_scale(uint32_t byte) {
    return __uint_as_float(byte == F8_NAN_BYTE ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// Two numbers as e4m3 codes, `lo` in the low byte (nearest, ties to even, magnitudes above 448 become 448).
__device__ __forceinline__ uint32_t f8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two codes as half-precision numbers (exact), the low byte's in the low half.
__device__ __forceinline__ uint32_t f8_to_f16x2(uint16_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
    return r;
}

// Two codes as numbers, the low byte's first.
__device__ __forceinline__ float2 f8_codes2(uint32_t two) {
    const uint32_t h = f8_to_f16x2((uint16_t)two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// A head's norm as the writers of the cache take it.  The reciprocal root of a mean square, to its last bits: codes flip where an
// entry lies near the middle of two, so a Newton step follows the approximation (not at infinity, where it would make 0 into NaN).
__device__ __forceinline__ float f8_inverse_root(float mean) {
    const float guess = rsqrtf(mean);
    return mean > 1e-30f && mean < INFINITY ? fmaf(0.5f * guess, fmaf(-mean * guess, guess, 1.f), guess) : guess;
}
// Finite entries beyond 2^60 or so have a sum of squares beyond the floats; times this power of two they do not, and the norm is
// the same without its epsilon, which is nothing beside them.
#define F8_NORM_DOWN 8.4703294725430034e-22f          // 2^-70

// Cos and sin of position * frequency, as every kernel makes them that writes this cache or rotates queries for it.  The angle is formed and
// brought to [-pi, pi] in 64 bits: in 32 its error is 2^-24 of the angle itself, 0.008 radians at position 131,072, against
// 2^-9 of a rounding to bfloat16.
__device__ __forceinline__ float2 f8_turn(int pos, float freq) {
    const double a = (double)pos * (double)freq;
    const double z = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
    const float zh = (float)z, zl = (float)(z - (double)zh);         // sin(zh + zl) = sin zh + zl cos zh, zl < 2^-23
    float s, c;
    sincosf(zh, &s, &c);
    return make_float2(fmaf(-s, zl, c), fmaf(c, zl, s));
}

// What the attention kernels over these pages are given.
struct F8AttnParams {
    const bf16* q;            // [tokens, q_stride]: query heads first in each row
    int64_t q_stride;
    bf16* out;                // [tokens, nq * d]
    const uint8_t* k_pages;   // [pages, nkv, P, d]
    const uint8_t* v_pages;
    const uint8_t* scales;    // [pages, nkv, P, 2]
    const int* block_table;   // [rows, table_stride]
    const int* page_base;     // [rows]: pages given back at the front of a row's table
    const int* row_start;     // [rows + 1]: a row's first token
    const int* row_pos;       // [rows]: tokens of the row in the cache before this step
    const int* tiles;         // [n_tiles, 2]: row, first token of the tile within the row
    const float* sink;        // [nq] or null: exp(sink_h) in the softmax denominator (no key, no value)
    int table_stride, nq, nkv, logP;
    AttnMask mask;            // attention_mask.cuh
    float scale_log2;         // softmax scale * log2(e)
};
