// Numbers of four bits in blocks of 32 that share a power of two, which gfx950 converts in hardware.
//
// A number is sign and magnitude: bit 3 the sign, bits 0..2 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A block's scale is a byte b
// and stands for 2^(b - 127): 4.25 bits a number.  b is the smallest that leaves the block's largest magnitude at most 7
// units (what is above 6 then rounds to 6), kept in 2..252, so that every value is a normal bf16 and none overflows; 255
// marks a block in which a number was infinite or NaN, and reads as NaN.  Of the thresholds between 6 (nothing cut) and 8
// (the exponent of the largest, nothing else) 7 leaves normal numbers least error: 11.2 % rms, against 11.5 at both ends.
// Values are exact in bf16: what is computed with them is what the same bf16 numbers would give.
//
// Pages.  The block of one (page, kv head, 32 channels) has 17 * page size bytes.
//   keys:   of each slot 16 bytes, byte i channels 2i (low half) and 2i + 1; then the slots' scales, slot s at place
//           16 (s / 16) + 4 (s % 4) + (s / 4) % 4 (a lane of the score's product takes slots s, s + 4, s + 8, s + 12: their
//           scales are then one word);
//   values: byte rows i = 0..15 of one byte a slot, channels i (low half) and i + 16: a byte belongs to one token, and
//           consecutive tokens of a channel lie side by side, as the operand of the weighted sum wants them; then the
//           slots' scales in order.
// Matrices.  [rows, K / 2] bytes, byte i numbers 2i (low half) and 2i + 1; scales [rows, K / 32 filled up to a multiple of 16].
#pragma once
#include "common.h"

namespace gb {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4Block = 32;
constexpr int kFp4BadScale = 255;

__host__ __device__ __forceinline__ size_t fp4_block_bytes(int page) { return (size_t)17 * page; }
__host__ __device__ __forceinline__ int fp4_key_scale_place(int slot) { return (slot & ~15) + 4 * (slot & 3) + ((slot >> 2) & 3); }

// the scale byte of a block whose largest magnitude has these bits (NaN compares above infinity as bits do)
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t largest) {
  const int e = (int)(largest >> 23);
  if (e == 255) return kFp4BadScale;
  const int b = e - 2 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(b < 2 ? 2 : b > 252 ? 252 : b);
}
// 2^(b - 127) as the conversions take it: they read the exponent's bits alone, whatever stands in the others, and those of 255 make NaN
__device__ __forceinline__ float fp4_unit(uint32_t b) { return __uint_as_float(b << 23); }
// of byte i of a word
__device__ __forceinline__ float fp4_unit_of(uint32_t w, int i) { return __uint_as_float(i < 3 ? w << (23 - 8 * i) : w >> 1); }

// eight numbers to a word, number i in bits 4i..4i+3: divided by the unit, to the nearest, ties to even, at most 6
__device__ __forceinline__ uint32_t fp4_pack8(const float (&x)[8], float unit) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], unit, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], unit, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], unit, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], unit, 3);
  return w;
}

// the eight numbers of a word, in bf16, exactly
__device__ __forceinline__ bf16x8 fp4_unpack8(uint32_t w, float unit) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight elements from memory; `wide`: they begin at a 16-byte word
__device__ __forceinline__ void load8(const bf16* p, bool wide, float (&x)[8]) {
  bf16x8 v;
  if (wide) v = *reinterpret_cast<const bf16x8*>(p);
  else
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
__device__ __forceinline__ void load8(const float* p, bool wide, float (&x)[8]) {
  if (wide) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ void store8(bf16* p, bool wide, const float (&x)[8]) {
  if (wide) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16)x[i];
    *reinterpret_cast<bf16x8*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (bf16)x[i];
  }
}
__device__ __forceinline__ void store8(float* p, bool wide, const float (&x)[8]) {
  if (wide) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
}

// A 32-bit operand of a product on the bf16 matrix cores: the sum of three bf16 numbers, the bits of the mantissa in three runs of
// eight.  The other operand is exact in bf16, so that the three products are exact and their sum is rounded in 32 bits alone.  A number
// that is not finite goes into the first term, the others being zero.
template <typename T> constexpr int kFp4Terms = std::is_same_v<T, float> ? 3 : 1;
__device__ __forceinline__ void fp4_terms(const float (&x)[8], bf16x8 (&out)[3]) {
  uint32_t t[3][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = __builtin_canonicalizef(x[i]);   // (the mark of a NaN may lie in the low bits)
    t[0][i] = __float_as_uint(v);
    const float left = v - __uint_as_float(t[0][i] & 0xffff0000u), rest = fabsf(v) < __builtin_inff() ? left : 0.f;
    t[1][i] = __float_as_uint(rest);
    t[2][i] = __float_as_uint(rest - __uint_as_float(t[1][i] & 0xffff0000u));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(t[k][2 * i + 1], t[k][2 * i], 0x07060302u);   // the upper halves
    __builtin_memcpy(&out[k], w, sizeof w);
  }
}
// Probabilities as two bf16 numbers: the upper eight bits of the mantissa, and the nearest to what is left, together
// off by at most 2^-16 of the number.
__device__ __forceinline__ void fp4_terms(const float (&x)[8], bf16x8 (&out)[2]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[1][i] = (bf16)(x[i] - __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u));
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
  __builtin_memcpy(&out[0], w, sizeof w);
}
__device__ __forceinline__ void fp4_terms(const float (&x)[8], bf16x8 (&out)[1]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) out[0][i] = (bf16)x[i];
}

}  // namespace gb
