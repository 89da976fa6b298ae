// Four-bit groups on gfx950 (MI355X): 32 values share a bf16 scale, a value is one of the eight levels below with a
// sign.  v_cvt_scalef32_pk_bf16_fp4 turns two codes of a word into two bf16, exactly, so that codes are MFMA operands after
// half an instruction a value, and the scales meet the fp32 sums of a group's products (weights, keys) or
// the other operand (values).
#pragma once

#include "uttt_device.h"

namespace uttt {

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// the eight codes of a word, the first in its lowest bits
__device__ __forceinline__ bf16x8 fp4_values(uint32_t w) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// element i of packed bf16 values
__device__ __forceinline__ float bf16_of(uint32_t pair, int i) {
  return __uint_as_float(i ? pair & 0xffff0000u : pair << 16);
}

__device__ __forceinline__ uint32_t bf16_bits(bf16 x) { return __builtin_bit_cast(uint16_t, x); }

// A group's scale from its largest magnitude; `fine`: every value is finite.
__device__ __forceinline__ bf16 fp4_scale(float largest, bool fine) {
  const bf16 s = static_cast<bf16>(largest * (1.f / 6.f));
  return !fine ? static_cast<bf16>(NAN) : to_f32(s) < 1.17549435e-38f ? static_cast<bf16>(0.f) : s;
}

// The codes of eight values under scale s, as a word.  The quotient is the correctly rounded one: with value and scale moved to
// where the scale is in [.5, 1), the rounded reciprocal's product and one correction give it (a remainder of one product is
// exact), at a third of a division's instructions.  v_cvt_scalef32_pk_fp4_f32 takes the nearest level, of two as near the one
// with an even index, and 6 for more; a negative 0 is made 0.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], float s) {
  const int up = -__builtin_amdgcn_frexp_expf(s);
  const float sn = __builtin_amdgcn_ldexpf(s, up), inverse = 1.f / sn;
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float xn = __builtin_amdgcn_ldexpf(x[j], up), near = xn * inverse;
    q[j] = fmaf(fmaf(-near, sn, xn), inverse, near);
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.f, 3);
  const uint32_t some = (w | w >> 1 | w >> 2) & 0x11111111u;  // nibbles with a magnitude
  w &= 0x77777777u | some << 3;
  return s > 0.f ? w : 0u;
}

// One fp32 value as bf16 parts that add up to it: three hold all 24 bits, two 16 (the last one rounded).
// Parts but the last are cut off, not rounded, so that none overflows; what is not finite is the first alone.
template <int PARTS>
__device__ __forceinline__ void bf16_parts(float x, bf16 (&p)[PARTS]) {
  if constexpr (PARTS == 1) {
    p[0] = static_cast<bf16>(x);
  } else {
    float rest = x;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const float cut = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
      p[i] = i == PARTS - 1 ? static_cast<bf16>(rest) : static_cast<bf16>(cut);
      rest -= cut;
      if (i == 0) rest = fabsf(x) < INFINITY ? rest : 0.f;
    }
  }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

}  // namespace uttt
