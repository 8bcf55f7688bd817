// Quantise to and from microscaled 4-bit weights (format in mx.hpp).
//
// quantise: the scale byte of a group is its largest magnitude's exponent less
// e2m1's own largest (2), in [0, 254]: 2^(floor(log2 max) - 2); each value
// divided by it rounds to the nearest code, ties to the even one, magnitudes
// above 6 to 6 (a group's largest lies in [4, 8) of its scale).  A group with an
// infinity or a NaN gets byte 255 and codes 0: it reads back as NaN.
// dequantise: code * scale, exact in f32, and in bf16 (past bf16's range an
// infinity).
// HBM-bound, one pass: a lane takes 8 values (16 bytes of bf16, 32 of f32), one
// word of codes; the four lanes of a group find its maximum by DPP moves, as
// integers, so that NaN compares largest.  A bank of 128 x 768 x 2048 bf16 weights: 81
// us, 6.3 TB/s, and 71 us back, 7.2.
#include <algorithm>

#include "mx.hpp"

namespace mlxr_moe {
namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

// How the values are reached: one by one (any alignment), by 16-byte vectors, or by
// such that keep no place in the caches, for arrays larger than the memory-side cache
// (256 MB), of which no reader after the kernel could find much there.  A bank of 403 MB
// there and back 184 us a pass with vectors, 166 with such loads, 152 with such stores
// too; smaller arrays stay where their reader finds them.
enum { kScalar, kVector, kStreamed };
template <int HOW, class V>
__device__ __forceinline__ V load16(const V* p) {
  if constexpr (HOW == kStreamed) return __builtin_nontemporal_load(p);
  return *p;
}
template <int HOW, class V>
__device__ __forceinline__ void store16(V* p, V v) {
  if constexpr (HOW == kStreamed)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

// 8 values from flat element e0 on, as f32.
template <bool BF16, int HOW>
__device__ __forceinline__ void load8(const void* w, int64_t e0, float (&v)[8]) {
  if constexpr (HOW != kScalar && BF16) {
    const u32x4_t u =
        load16<HOW>(reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(w) + e0));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(u[j] << 16);
      v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  } else if constexpr (HOW != kScalar) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(w) + e0);
    const f32x4_t a = load16<HOW>(p), b = load16<HOW>(p + 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (BF16)
        v[j] = bf16_to_f32(static_cast<const uint16_t*>(w)[e0 + j]);
      else
        v[j] = static_cast<const float*>(w)[e0 + j];
    }
  }
}

template <bool BF16, int HOW>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* __restrict__ w, int64_t n,
                                                          uint32_t* __restrict__ wq,
                                                          uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t e0 = i * 8;
  if (e0 >= n) return;  // whole groups: 32 divides n, and a group its wave
  float v[8];
  load8<BF16, HOW>(w, e0, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  top = max(top, dpp_u<0xB1>(top));  // lane ^ 1
  top = max(top, dpp_u<0x4E>(top));  // lane ^ 2
  const uint32_t ex = top >> 23;
  const bool finite = ex != 255;
  const uint32_t byte = finite ? (ex > 2 ? ex - 2 : 0) : 255u;
  const float sc = mx_scale(finite ? byte : 127u);
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], sc, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], sc, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], sc, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], sc, 3);
  wq[i] = finite ? word : 0u;
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

template <bool OUT_BF16, int HOW>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* __restrict__ wq,
                                                            const uint8_t* __restrict__ scales,
                                                            int64_t n, void* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t e0 = i * 8;
  if (e0 >= n) return;
  const uint32_t w = wq[i];
  const float sc = mx_scale(scales[i >> 2]);
  if constexpr (OUT_BF16) {
    const u32x4_t v = __builtin_bit_cast(u32x4_t, mx_weights(w, sc));
    uint16_t* o = static_cast<uint16_t*>(out) + e0;
    if constexpr (HOW != kScalar) {
      store16<HOW>(reinterpret_cast<u32x4_t*>(o), v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[2 * j] = (uint16_t)v[j], o[2 * j + 1] = (uint16_t)(v[j] >> 16);
    }
  } else {
    const mx_f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0);
    const mx_f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
    const mx_f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2);
    const mx_f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
    float* o = static_cast<float*>(out) + e0;
    if constexpr (HOW != kScalar) {
      store16<HOW>(reinterpret_cast<f32x4_t*>(o), f32x4_t{a.x, a.y, b.x, b.y});
      store16<HOW>(reinterpret_cast<f32x4_t*>(o + 4), f32x4_t{c.x, c.y, d.x, d.y});
    } else {
      const float v[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[j];
    }
  }
}

// elements per launch (a grid holds under 2^32 threads)
constexpr int64_t kLaunchElems = (int64_t)1 << 34;

// how to reach an array of `bytes` at p
int how(const void* p, int64_t bytes) {
  if (reinterpret_cast<uintptr_t>(p) & 15) return kScalar;
  return bytes > ((int64_t)256 << 20) ? kStreamed : kVector;
}

#define MLXR_MX_HOW(CALL, BF, h) \
  do {                           \
    if ((h) == kStreamed)        \
      CALL(BF, kStreamed);       \
    else if ((h) == kVector)     \
      CALL(BF, kVector);         \
    else                         \
      CALL(BF, kScalar);         \
  } while (0)

}  // namespace

hipError_t launch_mx_quantize(const void* w, bool w_bf16, int64_t n, uint32_t* wq,
                              uint8_t* scales, hipStream_t s) {
  const int64_t es = w_bf16 ? 2 : 4;
  for (int64_t at = 0; at < n; at += kLaunchElems) {
    const int64_t m = std::min(n - at, kLaunchElems);
    const char* src = static_cast<const char*>(w) + at * es;
    const dim3 grid((unsigned)((m / 8 + 255) / 256));
    uint32_t* q = wq + at / 8;
    uint8_t* sc = scales + at / kMxGroup;
    const int h = how(src, n * es);
#define MLXR_MX_CALL(BF, H) mx_quantize_kernel<BF, H><<<grid, 256, 0, s>>>(src, m, q, sc)
    if (w_bf16)
      MLXR_MX_HOW(MLXR_MX_CALL, true, h);
    else
      MLXR_MX_HOW(MLXR_MX_CALL, false, h);
#undef MLXR_MX_CALL
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_mx_dequantize(const uint32_t* wq, const uint8_t* scales, int64_t n, void* out,
                                bool out_bf16, hipStream_t s) {
  const int64_t es = out_bf16 ? 2 : 4;
  for (int64_t at = 0; at < n; at += kLaunchElems) {
    const int64_t m = std::min(n - at, kLaunchElems);
    char* dst = static_cast<char*>(out) + at * es;
    const dim3 grid((unsigned)((m / 8 + 255) / 256));
    const uint32_t* q = wq + at / 8;
    const uint8_t* sc = scales + at / kMxGroup;
    const int h = how(dst, n * es);
#define MLXR_MX_CALL(BF, H) mx_dequantize_kernel<BF, H><<<grid, 256, 0, s>>>(q, sc, m, dst)
    if (out_bf16)
      MLXR_MX_HOW(MLXR_MX_CALL, true, h);
    else
      MLXR_MX_HOW(MLXR_MX_CALL, false, h);
#undef MLXR_MX_CALL
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
#undef MLXR_MX_HOW

}  // namespace mlxr_moe
