// mx_device.h -- device helpers of the MXFP4 operators.
#pragma once

#include "moe_device.h"

namespace gxmoe {

// The scale byte of a block of 32 whose largest magnitude has the bits `top`
// (sign cleared): 2^(floor(log2 max) - 2), so that the largest value lies in
// [4, 8) of the scale, where e2m1 ends at 6 (values above are 6).  At least
// 2^-126, the smallest whose fp32 form is a normal number; 255 where the block
// holds an infinity or NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t field = top >> 23;
  return field == 255u ? 255u : field < 3u ? 1u : field - 2u;
}

// Eight values over 2^(code - 127), rounded to the nearest e2m1 (ties to the
// even code, what lies above 6 to 6), the first in the lowest nibble; 0 for
// code 255, whose values are NaN whatever the nibbles say.
__device__ __forceinline__ uint32_t mx_pack8(const float (&v)[8], uint32_t code) {
  const float scale = __uint_as_float(code << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  return code == 255u ? 0u : r;
}

__device__ __forceinline__ uint32_t mx_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Clamped SwiGLU of one (gate, up) pair, NaN kept (a minimum would drop it):
// (up + 1) * gate * sigmoid(alpha * gate), with the hardware's exponential and
// reciprocal, each within one unit of fp32's last place; a sigmoid below 2^-126 is 0, as that reciprocal of it is.  The IEEE division and the polynomial exponential
// of gx_swiglu are five times the instructions, 16 us of a tile of 256 x 256.
__device__ __forceinline__ float mx_swiglu(float g, float u, float alpha, float limit) {
  g = g > limit ? limit : g;
  u = u > limit ? limit : u;
  u = u < -limit ? -limit : u;
  const float e = __builtin_amdgcn_exp2f(g * (alpha * -1.44269504088896340736f));
  return (u + 1.0f) * (g * __builtin_amdgcn_rcpf(1.0f + e));
}

}  // namespace gxmoe
