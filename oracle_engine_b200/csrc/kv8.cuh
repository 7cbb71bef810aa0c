// The 8-bit form of the paged key/value cache, shared by the kernels that write and read it.
//
// A row (one token's key or value of one KV head, HD values) is kept as HD codes of 8 bits and one float32 scale:
//   codes  [pages][2][KVH][64][HD]     int8, or e4m3
//   scales [pages][2][KVH][64]
// With a = the row's largest magnitude and c the largest code (127, or 448 for e4m3)
//   code = row * c / a rounded to the nearest code, ties to even;   scale = a / c rounded to float32;   the row reads as code * scale.
// The row is what a 16-bit cache would hold: the projected value, or the key turned by its position and rounded ONCE to bfloat16.
// Everything is then exact up to the two roundings above.  With x = x' 2^i and a = a' 2^j, x' and a' of 8 bits, the quotient x c / a
// differs from a border t between two codes by (x' c 2^k - t a') / a', a fraction with the denominator 2^k' a': it is t, or off it by
// 2^-16 of itself or more.  A float32 product with the rounded c / a is within 2^-22 of the quotient, and a value within
// 2^-19 of one of 12 bits, as borders are, is taken for that one: so it lies on the quotient's side of every border, or on it.  Codes
// and scales therefore do not depend on which kernel wrote them.
// A row with an infinite or undefined value gets codes 0 and an undefined scale: it reads as undefined, and codes are always numbers.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#define OE_KV_BF16 0
#define OE_KV_INT8 1
#define OE_KV_E4M3 2

// a * c - b * s rounded once to bfloat16.  Two float32 operations are within 2^-23 of the magnitudes they add; only a sum that near to the
// border between two bfloat16 is taken apart: the two products into a float32 and its error each, the sum likewise, and what is left
// over beside a float32 sum on the border settles it.
__device__ __noinline__ uint32_t kv8_turned_near(float a, float c, float b, float s) {
    const float p = __fmul_rn(a, c), ep = __fmaf_rn(a, c, -p);
    const float q = -__fmul_rn(b, s), eq = -__fmaf_rn(b, s, q);
    const float t = __fadd_rn(p, q), z = __fsub_rn(t, p);
    const float et = __fadd_rn(__fsub_rn(p, __fsub_rn(t, z)), __fsub_rn(q, z));
    const float rest = __fadd_rn(et, __fadd_rn(ep, eq));
    const float hi = __fadd_rn(t, rest), y = __fsub_rn(hi, t);
    const float lo = __fadd_rn(__fsub_rn(t, __fsub_rn(hi, y)), __fsub_rn(rest, y));
    const uint32_t u = __float_as_uint(hi);
    if ((u & 0xffffu) == 0x8000u && lo != 0.f) return ((lo > 0.f) == (hi > 0.f)) ? (u >> 16) + 1u : u >> 16;
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi));
}
__device__ __forceinline__ uint32_t kv8_turned_bits(float a, float c, float b, float s) {
    const float q = __fmul_rn(b, s), hi = __fmaf_rn(a, c, -q);
    const uint32_t u = __float_as_uint(hi);
    const float border = __uint_as_float((u & 0xffff0000u) | 0x8000u);
    // (fabsf(hi) + fabsf(q) bounds |a c| as well: 2^-22 of it is more than either operation's error)
    if (!(fabsf(hi - border) > 2.38418579e-7f * (fabsf(hi) + fabsf(q)))) return kv8_turned_near(a, c, b, s);
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi));
}
__device__ __forceinline__ float kv8_from_bits(uint32_t b) { return __uint_as_float(b << 16); }

// What a row's codes are made from, of its largest magnitude as bfloat16 bits without the sign (an undefined value is the largest).
struct Kv8Row {
    float pre, by;         // a code is x * pre * by: pre a power of two that keeps c / (a pre) within float32's range
    float scale;
    bool bad;
};
template <int KIND>
__device__ __forceinline__ Kv8Row kv8_row(uint32_t max_bits) {
    constexpr float C = KIND == OE_KV_INT8 ? 127.f : 448.f;
    Kv8Row r;
    const float a = kv8_from_bits(max_bits);
    r.bad = max_bits >= 0x7f80u;
    r.pre = a >= 1.26765060e30f ? 5.42101086e-20f : a < 7.88860905e-31f ? 1.84467441e19f : 1.f;      // 2^100: 2^-64; below 2^-100: 2^64
    r.by = a > 0.f ? __fdiv_rn(C, a * r.pre) : 0.f;
    r.scale = r.bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, C);
    if (r.bad) r.by = 0.f;
    return r;
}
template <int KIND>
__device__ __forceinline__ float kv8_quotient(const Kv8Row& r, uint32_t bits) {
    const float y = __fmul_rn(__fmul_rn(kv8_from_bits(bits), r.pre), r.by);
    const uint32_t u = __float_as_uint(y) + 16u;            // within 16 of a multiple of 2^11 in the last place: that multiple
    const uint32_t v = (u & 0x7ffu) <= 32u ? u & 0xfffff800u : u - 16u;
    return r.bad ? 0.f : __uint_as_float(v);
}
template <int KIND>
__device__ __forceinline__ uint32_t kv8_code(const Kv8Row& r, uint32_t bits) {
    const float x = kv8_quotient<KIND>(r, bits);
    if (KIND == OE_KV_INT8) return (uint32_t)(__float2int_rn(x) & 0xff);
    return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
// Four codes of consecutive values, two to a word of `bits`, the first in the lowest byte.
template <int KIND>
__device__ __forceinline__ uint32_t kv8_codes4(const Kv8Row& r, uint32_t b01, uint32_t b23) {
    const float x0 = kv8_quotient<KIND>(r, b01 & 0xffffu), x1 = kv8_quotient<KIND>(r, b01 >> 16);
    const float x2 = kv8_quotient<KIND>(r, b23 & 0xffffu), x3 = kv8_quotient<KIND>(r, b23 >> 16);
    if (KIND == OE_KV_INT8) {
        // 1.5 * 2^23 + x, rounded to nearest even as the sum is: its lowest byte is the code
        const uint32_t i0 = __float_as_uint(__fadd_rn(x0, 12582912.f)), i1 = __float_as_uint(__fadd_rn(x1, 12582912.f));
        const uint32_t i2 = __float_as_uint(__fadd_rn(x2, 12582912.f)), i3 = __float_as_uint(__fadd_rn(x3, 12582912.f));
        return __byte_perm(__byte_perm(i0, i1, 0x0040u), __byte_perm(i2, i3, 0x0040u), 0x5410u);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x2, x3), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

__device__ __forceinline__ uint32_t kv8_prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// Codes as two float16 (every code is a float16 exactly).  int8 codes come with their sign bits turned (kv8_words): bits
// 0x6400 | (code + 128) are 1,152 + code.  `lo`: the first of the two bytes of x, 0 or 2.
template <int KIND>
__device__ __forceinline__ uint32_t kv8_word(uint32_t w) { return KIND == OE_KV_INT8 ? w ^ 0x80808080u : w; }
template <int KIND>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t x, int lo) {
    uint32_t d;
    if (KIND == OE_KV_INT8) {
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(kv8_prmt(x, 0x64646464u, lo == 0 ? 0x4140u : 0x4342u)), "r"(0x64806480u));
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(lo == 0 ? x : x >> 16));
    }
    return d;
}
// A query row as float16: multiplied by the power of two that brings its largest magnitude into [1, 2), so that nothing leaves
// float16's range and 11 bits are kept of every value within 2^-14 of the largest.  `up`: the inverse, for the scores.
__device__ __forceinline__ float kv8_row_factor(float largest, float* up) {
    int e = (int)(__float_as_uint(largest) >> 23) & 0xff;
    e = min(max(e, 1), 253);
    *up = __uint_as_float((uint32_t)e << 23);
    return __uint_as_float((uint32_t)(254 - e) << 23);
}
// The power of two above a row's scale (a scale that is no number counts as none).
__device__ __forceinline__ float kv8_above(float scale) {
    const uint32_t u = __float_as_uint(fmaxf(scale, 0.f));
    return __uint_as_float((u & 0x7f800000u) + 0x00800000u);
}
__device__ __forceinline__ float kv8_inverse(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }
