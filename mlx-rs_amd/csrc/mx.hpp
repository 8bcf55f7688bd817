// Microscaled 4-bit weights and 8-bit activations (modes "mxfp4", "mxfp8"): device
// helpers.
//
// A group of 32 values of a row shares one scale byte b, the power of two
// 2^(b - 127); b = 255 is NaN.  A value is a 4-bit e2m1 code -- sign, two
// exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- times the scale
// (the concrete format MXFP4 of the OCP Microscaling Formats specification,
// v1.0).  Eight codes to a 32-bit word, the first lowest.  Every such weight is a
// bf16 value exactly while the product stays in bf16's range (b < 253), so the
// products below multiply the same weights whichever kernel runs.
//
// Mode "mxfp8" (MXFP8 of the same) has 8-bit e4m3 codes -- sign, four exponent bits
// of bias 7, three mantissa bits, magnitudes up to 448 -- four to a word, and the
// same scales.
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

// ---- mode "mxfp8"
// The scale byte of a group whose largest magnitude has the bits `top`: its exponent
// less e4m3's own largest (8), at least 0; 255 where an infinity or a NaN is among
// them (integers compare NaN largest).
__device__ __forceinline__ uint32_t mx8_byte(uint32_t top) {
  const uint32_t ex = top >> 23;
  return ex == 255 ? 255u : ex > 8 ? ex - 8 : 0u;
}
// The codes of a and b, low byte first, under that scale: the nearest ones (ties to
// the even code), magnitudes above 448 to 448; 0 under 255.  The division by the
// power of two is exact.
__device__ __forceinline__ uint32_t mx8_pair(float a, float b, uint32_t byte) {
  if (byte == 255) return 0;
  const float inv = __uint_as_float((254u - byte) << 23);
  a = __builtin_amdgcn_fmed3f(a * inv, -448.0f, 448.0f);
  b = __builtin_amdgcn_fmed3f(b * inv, -448.0f, 448.0f);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
// 8 values of a lane, a group being four neighbouring lanes': their codes and the
// group's scale byte.
__device__ __forceinline__ uint32_t mx8_group8(const float (&v)[8], uint2& q) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
  const uint32_t byte = mx8_byte(top);
  q.x = mx8_pair(v[0], v[1], byte) | (mx8_pair(v[2], v[3], byte) << 16);
  q.y = mx8_pair(v[4], v[5], byte) | (mx8_pair(v[6], v[7], byte) << 16);
  return byte;
}
// The value of a scale byte, exactly.
__device__ __forceinline__ float mx8_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

}  // namespace mlxr_moe
