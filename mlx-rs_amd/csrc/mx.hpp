// Microscaled 4-bit weights (mode "mxfp4"): device helpers.
//
// A group of 32 values of a row shares one scale byte b, the power of two
// 2^(b - 127); b = 255 is NaN.  A value is a 4-bit e2m1 code -- sign, two
// exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- times the scale
// (the concrete format MXFP4 of the OCP Microscaling Formats specification,
// v1.0).  Eight codes to a 32-bit word, the first lowest.  Every such weight is a
// bf16 value exactly while the product stays in bf16's range (b < 253), so the
// products below multiply the same weights whichever kernel runs.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace mlxr_moe {

constexpr int kMxGroup = 32;

typedef __bf16 mx_bf16x2_t __attribute__((ext_vector_type(2)));
typedef float mx_f32x2_t __attribute__((ext_vector_type(2)));

// The scale operand of the conversions below, which read its exponent field: 0
// is 2^-127 and 255 is NaN there (all 256 bytes x 16 codes checked on the device
// against the format's definition).
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// The eight weights of one word as an MFMA operand, in order.
__device__ __forceinline__ bf16x8_t mx_weights(uint32_t w, float scale) {
  u32x4_t r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  return as_bf16x8(r);
}

// The gated products' activation in f32, rounded to bf16 once, where the second
// product takes it up (the affine modules round after every op, as the
// reference's bf16 chain does, and lose a bit more: y of a c2 bank is off by 2.3
// parts in a thousand here and by 4.2 so, its own rounding 1.7 of them).
//   swiglu: g sigmoid(g) u
//   geglu:  0.5 g (1 + tanh(y)) u = g sigmoid(2 y) u,  y = c (g + k g^3), with the
//           constants as the reference's bf16 chain holds them
// The sigmoid from the hardware exp2 and reciprocal, about an ulp each.
__device__ __forceinline__ float mx_act(int act, float g, float u) {
  float y = g;
  if (act == kActGeglu) {
    const float k = 0.044677734375f, c = 0.796875f;
    y = 2.0f * c * g * __builtin_fmaf(k * g, g, 1.0f);
  }
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * y);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}
__device__ __forceinline__ uint16_t mx_bf16(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}

}  // namespace mlxr_moe
