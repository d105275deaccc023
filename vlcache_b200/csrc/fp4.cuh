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

#include "common.cuh"

namespace vlc {
namespace fp4 {

constexpr int HD = 128;
constexpr int GROUP = 16;
constexpr int CODE_BYTES = HD / 2;
constexpr int SCALE_BYTES = HD / GROUP;
constexpr int ROW_BYTES = CODE_BYTES + SCALE_BYTES;

// Offset of a head's piece of a page, and of a row's codes and scales in it.
__host__ __device__ __forceinline__ int64_t head_offset(int64_t page, int num_kv_heads, int head, int block_size) {
  return (page * num_kv_heads + head) * ((int64_t)block_size * ROW_BYTES);
}
__host__ __device__ __forceinline__ int code_offset(int row) { return row * CODE_BYTES; }
__host__ __device__ __forceinline__ int scale_offset(int row, int block_size) {
  return block_size * CODE_BYTES + row * SCALE_BYTES;
}

// Eight floats to eight e2m1 codes (nearest even, magnitudes above 6 become 6).
__device__ __forceinline__ uint32_t encode8(const float (&y)[8]) {
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

__device__ __forceinline__ float scale_f32(uint32_t byte) {
  const uint32_t h = scales2_f16(byte & 0xff);
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffff)));
}

// The scale byte of a group whose largest magnitude is amax (NaN for NaN).
__device__ __forceinline__ uint32_t encode_scale(float amax) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(__fdiv_rn(amax, 6.f)));
  return r & 0xff;
}

// Largest magnitude of eight floats, as its bit pattern: integers order magnitudes as floats do
// and put every NaN above infinity, so a NaN survives the maximum.
__device__ __forceinline__ uint32_t absmax8_bits(const float (&y)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
  return m;
}

// Codes of eight elements of a group with the given scale byte.  The quotient is the correctly
// rounded one: a tie between two codes is then a tie in the arithmetic too.
__device__ __forceinline__ uint32_t quantise8(const float (&y)[8], uint32_t scale_byte) {
  const float s = scale_f32(scale_byte);
  if (s == 0.f) return 0;
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = __fdiv_rn(y[i], s);
  return encode8(t);
}

}  // namespace fp4
}  // namespace vlc
