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

}  // namespace mlxr_moe
