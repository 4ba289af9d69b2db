// tp_codes.h -- registers of packed fp16 and the decoded angles and values of page codes, as
// the attention kernels use them.
#pragma once

#include "tp_common.h"

namespace tp {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half8v as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(half8v, v);
}

__device__ __forceinline__ uint32_t pack_h2(half2v v) { return __builtin_bit_cast(uint32_t, v); }

__device__ __forceinline__ half2v lo_lo(uint32_t w) {
  const f16 r = __builtin_bit_cast(f16, (uint16_t)(w & 0xffffu));
  return half2v{r, r};
}
__device__ __forceinline__ half2v hi_hi(uint32_t w) {
  const f16 r = __builtin_bit_cast(f16, (uint16_t)(w >> 16));
  return half2v{r, r};
}

// (cos, sin) of a code's decoded angle, rounded to fp16 and packed: the
// reference's fp32 angle (code_angle, decoder.py:37-55) through accurate fp32
// cosf / sinf.  At half a turn the reference's sin(f32(pi)) is -8.7e-8, whose
// fp16 rounding -5.96e-8 is not zero, so an inf radius decodes to -inf there
// as in the reference (decoder.py:57-67); the hardware sine in revolutions
// returns an exact 0 at half a turn, which would turn that product into NaN.
// No code of 2, 4 or 8 bits has a cosine or sine that rounds to fp16 zero.
__device__ __forceinline__ uint32_t make_cs(uint32_t code, int bits) {
  const float th = code_angle(code, bits);
  const half2v cs = {(f16)cosf(th), (f16)sinf(th)};
  return pack_h2(cs);
}

// Four int8 codes -> two exact fp16 pairs: bias the byte into the mantissa of
// 1024.0 (0x64xx) after flipping its sign bit, then subtract 1152.
__device__ __forceinline__ void i8x4_to_f16(uint32_t w, half2v& lo, half2v& hi) {
  const uint32_t x = w ^ 0x80808080u;
  const uint32_t a = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
  const uint32_t b = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
  const half2v bias = {(f16)1152.0f, (f16)1152.0f};
  lo = __builtin_bit_cast(half2v, a) - bias;
  hi = __builtin_bit_cast(half2v, b) - bias;
}

}  // namespace tp
