// The 4-bit KV cache: its page layout and its conversions.
//
// A head's row of 128 dims is 8 groups of 16.  A group holds one e4m3 scale s and 16 e2m1 codes
// (two per byte, the even dim in the low nibble); with g a power of two per cache
//   s = e4m3(min(max|x / g| / 6, 448)),  code = e2m1(x / g / s),  value = g * s * code,
// every conversion rounded to nearest even (codes are 0 where s is 0; a NaN makes its group's s
// NaN).  6 is the largest e2m1 magnitude.  e2m1 has 2 significant bits and e4m3 has 4, so a value
// has at most 6 and the powers of two between 2^-10 and 2^11: it is exact in f16 and in bf16, and
// dequantising never rounds.
//
// One layer's K (or V) page is [num_kv_heads][block_size * 64 code bytes | block_size * 8 scale
// bytes]: 72 bytes per row and head, the rows of a head consecutive, so that a run of keys of one
// head is one contiguous piece of codes and one of scales.
#pragma once

#include <cmath>

#include "common.cuh"

namespace vlc {
namespace fp4 {

constexpr int HD = 128;
constexpr int GROUP = 16;
constexpr int CODE_BYTES = HD / 2;
constexpr int SCALE_BYTES = HD / GROUP;
constexpr int ROW_BYTES = CODE_BYTES + SCALE_BYTES;
constexpr int MAX_BLOCK = 1 << 20;  // a head's piece of a page stays within 32-bit offsets

// Whether g may be a cache's power of two: 2^-64 .. 2^64.
inline bool power_of_two(float g) {
  int e;
  return std::isfinite(g) && g > 0.f && std::frexp(g, &e) == 0.5f && e >= -63 && e <= 65;
}

// Offset of a head's piece of a page, and of a row's codes and scales in it.
__host__ __device__ __forceinline__ int64_t head_offset(int64_t page, int num_kv_heads, int head, int block_size) {
  return (page * num_kv_heads + head) * ((int64_t)block_size * ROW_BYTES);
}
__host__ __device__ __forceinline__ int code_offset(int row) { return row * CODE_BYTES; }
__host__ __device__ __forceinline__ int scale_offset(int row, int block_size) {
  return block_size * CODE_BYTES + row * SCALE_BYTES;
}

// Eight codes to four f16 pairs: pair i holds byte i's low nibble (low half) and high nibble.
__device__ __forceinline__ void decode8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// Two e4m3 bytes (low byte first) to an f16 pair.
__device__ __forceinline__ uint32_t scales2_f16(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}

// Eight bf16 values (a uint4) as four packed fp32 pairs.
__device__ __forceinline__ void unpack8(const uint4& w, uint64_t (&f)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
// And back, rounded to nearest even.
__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_unpack(f[i], lo, hi);
    u[i] = pack_bf16x2(lo, hi);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Rotate-half pairs: x1 = x1 c - x2 s, x2 = x2 c + x1 s, every product and sum rounded by itself.
// The products are packed, the sums are not: the assembler joins a packed product and a packed sum
// into one packed fma in spite of their .rn (46 % of random sums differed), but leaves these.
__device__ __forceinline__ void rotate8(uint64_t (&x1)[4], uint64_t (&x2)[4], const uint64_t (&c)[4],
                                        const uint64_t (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a0, a1, b0, b1, e0, e1, f0, f1;
    f2_unpack(f2_mul(x1[i], c[i]), a0, a1);
    f2_unpack(f2_mul(x2[i], s[i]), b0, b1);
    f2_unpack(f2_mul(x2[i], c[i]), e0, e1);
    f2_unpack(f2_mul(x1[i], s[i]), f0, f1);
    x1[i] = f2_pack(__fsub_rn(a0, b0), __fsub_rn(a1, b1));
    x2[i] = f2_pack(__fadd_rn(e0, f0), __fadd_rn(e1, f1));
  }
}

// ---- quantising bf16 rows: a group's largest magnitude, its scale byte, its codes

// Largest of eight bf16 magnitudes, as 15 bits: integers order magnitudes as floats do and put
// every NaN above infinity, so a NaN survives the maximum.
__device__ __forceinline__ uint32_t absmax8(const uint4& w) {
  const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                              __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  return max(m & 0xffffu, m >> 16);
}

// The scale byte of a group with that largest magnitude, after division by g (1 / g given; NaN for
// NaN).  The product with the fp32 next to 1/6 rounds to e4m3 as the quotient by 6 does: it is off
// by at most 2^-23 of it; a magnitude of 8 bits is a tie (6 times a value halfway between two
// scales) or 2^-9 away from one; and at the 126 ties the product is exact.
__device__ __forceinline__ uint32_t encode_scale(uint32_t top, float inv_g) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
      : "=h"(r)
      : "f"(0.f), "f"(__uint_as_float(top << 16) * inv_g * (1.f / 6.f)));
  return r & 0xff;
}

// 1 / (g s) of a scale byte; 0 for a scale of 0, whose codes are 0.
__device__ __forceinline__ float inverse_scale(uint32_t byte, float inv_g) {
  const uint32_t h = scales2_f16(byte & 0xff);
  const float s = __half2float(__ushort_as_half((unsigned short)(h & 0xffff)));
  return s == 0.f ? 0.f : __fdividef(inv_g, s);
}

// Codes of eight values of a group, given 1 / (g s).  x / (g s) is wanted rounded to e2m1 as the
// exact quotient is.  A quotient of 8 by 4 bits either is a tie of e2m1 (0.25 .. 5, multiples of
// 2^-2) or differs from every tie by 2^-8 of it; so it is first put on the grid of 2^-11 by adding
// and taking away 1.5 * 2^12, where ties are exact and the product's error of some 2^-22 is gone.
__device__ __forceinline__ uint32_t quantise8(const uint4& w, float inv) {
  constexpr float GRID = 1.5f * 4096.f;
  const uint64_t big = f2_pack(GRID, GRID), minus = f2_pack(-GRID, -GRID);
  const uint64_t inv2 = f2_pack(inv, inv);
  uint64_t x[4];
  unpack8(w, x);
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(f2_add(f2_fma(x[i], inv2, big), minus), y[2 * i], y[2 * i + 1]);
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}

}  // namespace fp4
}  // namespace vlc
