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
// 2^-16 of itself or more.  A float32 product with the rounded c / a is within 2^-22 of the quotient; rounded to 18 bits (Veltkamp's
// splitting) it is the border itself where the quotient is one, and on the quotient's side of it where not.  Codes and scales
// therefore do not depend on which kernel wrote them.
// A row with an infinite or undefined value gets codes 0 and an undefined scale: it reads as undefined, and codes are always numbers.
#pragma once
#include "common.cuh"
#include <atomic>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

// On which devices a kernel's attributes have been set (they are a device's; setting them again does no harm).
struct Kv8Devices {
    std::atomic<unsigned long long> bits{0};
    static int current() { int d = 0; return cudaGetDevice(&d) == cudaSuccess && d < 64 ? d : -1; }
    bool first() const { const int d = current(); return d < 0 || !(bits.load(std::memory_order_acquire) >> d & 1ull); }
    void done() { const int d = current(); if (d >= 0) bits.fetch_or(1ull << d, std::memory_order_release); }
};

#define OE_KV_BF16 0
#define OE_KV_INT8 1
#define OE_KV_E4M3 2

// What an entry point of these kernels is told, as the host packs it (one argument to convert instead of thirty); a field that an entry
// point does not use is 0.
struct Kv8Call {
    __nv_bfloat16* out;            // [n_tokens, H*HD]
    const __nv_bfloat16* qkv;      // [n_tokens, (H + 2 KVH) HD], or queries only; rows of `stride`
    long long stride;
    const float *cos_tab, *sin_tab;
    void* cache;                   // a cache entry's codes, or its bfloat16 rows
    float* scales;
    long long n_pages;
    const int *tables, *cu_q, *seq_start, *seq_qlen, *tok_seq, *tok_pos;
    const int *members, *first, *pages, *seq_pages;     // of prefixes
    float *part_o, *part_ml;       // [n_tokens * H, parts, HD], [n_tokens * H, parts, 2]; parts: shares, or splits
    cudaStream_t stream;
    int bytes;                     // of this struct
    int kind, write, max_pages, n_seqs, n_tokens, max_qlen, H, KVH, window, warps, cluster, ordered, shares, mt, splits, n_groups, n_members, ahead;
    int n_positions, n_tables;     // that the angles and (for the write) the page tables are there for
    float scale;
};
static_assert(sizeof(Kv8Call) == 21 * 8 + 22 * 4, "as the host packs it");

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
__device__ __forceinline__ uint32_t kv8_turned_fast(float a, float c, float b, float s, bool& near) {
    const float q = __fmul_rn(b, s), hi = __fmaf_rn(a, c, -q);
    const float border = __uint_as_float((__float_as_uint(hi) & 0xffff0000u) | 0x8000u);
    // (either operation's error is at most 2^-24 of its result: together less than 1.2e-7 > 2^-23 of the two)
    near = near || !(fabsf(hi - border) > 1.2e-7f * (fabsf(hi) + fabsf(q)));
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi));
}
__device__ __forceinline__ float kv8_from_bits(uint32_t b) { return __uint_as_float(b << 16); }

// N pairs (x0, x1) of a row, two bfloat16 to a word of lo and of hi, turned by cs and sn: x0 cs - x1 sn and x0 sn + x1 cs.
template <int N>
__device__ __forceinline__ void kv8_turn(uint32_t (&lo)[N / 2], uint32_t (&hi)[N / 2], const float (&cs)[N], const float (&sn)[N]) {
    uint32_t nl[N / 2], nh[N / 2];
    bool near = false;
#pragma unroll
    for (int j = 0; j < N / 2; j++) {
        const float x0 = kv8_from_bits(lo[j]), y0 = __uint_as_float(lo[j] & 0xffff0000u), x1 = kv8_from_bits(hi[j]), y1 = __uint_as_float(hi[j] & 0xffff0000u);
        nl[j] = kv8_turned_fast(x0, cs[2 * j], x1, sn[2 * j], near) | kv8_turned_fast(y0, cs[2 * j + 1], y1, sn[2 * j + 1], near) << 16;
        nh[j] = kv8_turned_fast(x0, sn[2 * j], -x1, cs[2 * j], near) | kv8_turned_fast(y0, sn[2 * j + 1], -y1, cs[2 * j + 1], near) << 16;
    }
    if (near) {
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            const float x0 = kv8_from_bits(lo[j]), y0 = __uint_as_float(lo[j] & 0xffff0000u), x1 = kv8_from_bits(hi[j]), y1 = __uint_as_float(hi[j] & 0xffff0000u);
            nl[j] = kv8_turned_near(x0, cs[2 * j], x1, sn[2 * j]) | kv8_turned_near(y0, cs[2 * j + 1], y1, sn[2 * j + 1]) << 16;
            nh[j] = kv8_turned_near(x0, sn[2 * j], -x1, cs[2 * j]) | kv8_turned_near(y0, sn[2 * j + 1], -y1, cs[2 * j + 1]) << 16;
        }
    }
#pragma unroll
    for (int j = 0; j < N / 2; j++) { lo[j] = nl[j]; hi[j] = nh[j]; }
}
// The largest magnitudes of two words' halves, as bfloat16 bits (an undefined value is the largest).
__device__ __forceinline__ uint32_t kv8_most(uint32_t a, uint32_t b) { return __vmaxu2(a, b & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t kv8_most(uint32_t a) { return max(a & 0xffffu, a >> 16); }

// From the bits of a row's largest magnitude: c / a for its codes, and its scale.  The words of a row that cannot be had that way
// are changed: to zero where there is no largest magnitude, and times 2^64 where c / a would leave float32's range.
template <int KIND, int N>
__device__ __forceinline__ float kv8_row(uint32_t max_bits, uint32_t (&words)[N], float* scale) {
    constexpr float C = KIND == OE_KV_INT8 ? 127.f : 448.f;
    float a = kv8_from_bits(max_bits);
    *scale = max_bits >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, C);
    if (max_bits >= 0x7f80u || max_bits == 0u) {
#pragma unroll
        for (int j = 0; j < N; j++) words[j] = 0u;
        return 0.f;
    }
    if (a < 7.88860905e-31f) {                              // 2^-100
        a *= 1.84467441e19f;                                // 2^64
#pragma unroll
        for (int j = 0; j < N; j++)
            words[j] = __float_as_uint(kv8_from_bits(words[j]) * 1.84467441e19f) >> 16 |
                       (__float_as_uint(__uint_as_float(words[j] & 0xffff0000u) * 1.84467441e19f) & 0xffff0000u);
    }
    return __fdiv_rn(C, a);
}
__device__ __forceinline__ float kv8_quotient(float x, float by) {
    const float y = __fmul_rn(x, by), t = __fmul_rn(y, 65.f);
    return __fsub_rn(t, __fsub_rn(t, y));
}
// The codes of two words' four values, the first in the lowest byte.
template <int KIND>
__device__ __forceinline__ uint32_t kv8_codes4(float by, uint32_t b01, uint32_t b23) {
    const float x0 = kv8_quotient(kv8_from_bits(b01), by), x1 = kv8_quotient(__uint_as_float(b01 & 0xffff0000u), by);
    const float x2 = kv8_quotient(kv8_from_bits(b23), by), x3 = kv8_quotient(__uint_as_float(b23 & 0xffff0000u), by);
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
// The same in an order that costs less: int8's first pair are the bytes 0 and 2, its second the bytes 1 and 3; e4m3's 0 and 1, and 2 and 3.
// (The shift is a product's upper half: shifts, permutes and logic share the pipe that conversions are bound by.)
template <int KIND>
__device__ __forceinline__ uint32_t kv8_first(uint32_t w) {
    if (KIND != OE_KV_INT8) return kv8_pair<KIND>(w, 0);
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((w & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
    return d;
}
template <int KIND>
__device__ __forceinline__ uint32_t kv8_second(uint32_t w) {
    return KIND == OE_KV_INT8 ? kv8_first<KIND>(__umulhi(w, 1u << 24)) : kv8_pair<KIND>(w, 2);
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
