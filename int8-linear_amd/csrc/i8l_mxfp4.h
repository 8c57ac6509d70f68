// Device pieces of the MXFP4 operators (OCP microscaling): E2M1 elements (1 sign, 2 exponent, 1
// mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two a byte with the even element in the low nibble,
// and one E8M0 scale 2^(byte - 127) for each 32 elements of a row, 255 meaning NaN.
#pragma once

#include "i8l_common.h"

namespace i8l {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int kMxBlock = 32;

// The E8M0 code of a block whose largest magnitude has the float bits `peak` (sign clear):
// floor(log2(peak)) - 2, so that peak / scale lies in [4, 8) and what is past 6 saturates; with
// `rounded`, peak is first rounded to E2M1's one mantissa bit, so that peaks from 1.75 * 2^e take
// the next scale and no element loses more than half a step.  Below 2^-125 the scale stays at
// 2^-127 (all-zero blocks too); a block with an infinity or a NaN gets the NaN scale.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t peak, int rounded) {
  const uint32_t e = (peak + (rounded ? 0x200000u : 0u)) >> 23;
  return peak >= 0x7f800000u ? 255u : max(e, 2u) - 2u;
}

// The largest of the four lanes of a quad, which hold a block of 32, 8 elements each.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)dpp_i<kQuadSwap1>((int)v));
  return max(v, (uint32_t)dpp_i<kQuadSwap2>((int)v));
}

// The codes of 8 elements as a word, element 0 in the low nibble: x / 2^(code - 127), rounded to
// nearest even and saturated at 6, by the scaled conversions (v_cvt_scalef32_pk_fp4_*; they take
// the scale as the float with that exponent field, 2^-127 for field 0; checked on gfx950 for every
// bf16 and fp16 and over random floats, at scales of both ends).  A NaN-scaled block holds zeros.
__device__ __forceinline__ uint32_t mx_codes8(const float (&y)[8], uint32_t code) {
  const float s = __uint_as_float(code << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], s, 3);
  return code == 255u ? 0u : r;
}

// The same for 8 packed bf16 or fp16 elements.
template <int DT>
__device__ __forceinline__ uint32_t mx_codes8(const uint4& v, uint32_t code) {
  const float s = __uint_as_float(code << 23);
  uint32_t r = 0;
  if constexpr (DT == I8L_BF16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(v2bf, v.x), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(v2bf, v.y), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(v2bf, v.z), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(v2bf, v.w), s, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(v2h, v.x), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(v2h, v.y), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(v2h, v.z), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(v2h, v.w), s, 3);
  }
  return code == 255u ? 0u : r;
}

// 2^(code - 127) as a float (a subnormal for code 0), NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t code) {
  return __uint_as_float(code == 0 ? 0x00400000u : code == 255u ? 0x7fc00000u : code << 23);
}

// The value of an E2M1 code.
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  const uint32_t m = c & 7;
  const float a = m < 4 ? 0.5f * m : m < 6 ? (float)m - 2.0f : 2.0f * m - 8.0f;
  return c & 8 ? -a : a;
}

}  // namespace i8l
