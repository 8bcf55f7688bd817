// The residual add with the RMSNorm behind it, and its gradients, on gfx950.
//
// Over rows x, residual [T, d] and a weight w [d]:
//   h = x + residual                (rounded to the residual's type: the stream)
//   r = 1 / sqrt(sum_j h_j^2 / d + eps)
//   y_j = w_j h_j r
// y in bf16, rounded once, or in mode "mxfp8": e4m3 codes with a power-of-two scale
// per 32 (mx.hpp), each the nearest of the value in f64.  With dy the gradient of y
// and dh what comes to h from elsewhere,
//   g_j  = dy_j w_j,  c = sum_j g_j h_j / d
//   dx_j = r (g_j - h_j r^2 c) + dh_j      (of x and of the residual alike)
//   dw_j = sum_t dy_tj h_tj r_t
// All sums in f32 (the weight gradient's over workgroups in f64), in fixed orders.
//
// HBM-bound: one pass over the rows, a row held in registers, by a wave (many rows)
// or by a workgroup of four (few rows, or wide ones), in 16-byte accesses; a form of the
// kernels takes them at any address and of any length, and rows of more than 16384 values
// or less than 8 go by single ones.  Measured: 8192 rows
// of 2048, f32 + bf16 to bf16 and codes, 33 us (4.6 TB/s); the gradients of 32768 of 2048 in
// f32 167 + 5 us (5.6 TB/s), of 1000 of 4096 in bf16 12 + 4; one row 2.3.  Rows of 2047 as
// those of 2048 (single values in place of their 16 bytes: 196 us against 104 forward, the
// gradients 217 against 127, 32768 rows in bf16).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "mx.hpp"
#include "nn.hpp"

namespace mlxr_moe {
namespace {

constexpr int kNT = 256;

// 16 bytes at any element
typedef f32x4_t f32x4_any __attribute__((aligned(4)));
typedef u32x4_t u32x4_any __attribute__((aligned(2)));

template <bool F32>
__device__ __forceinline__ float load1(const void* p, int64_t e) {
  if constexpr (F32)
    return static_cast<const float*>(p)[e];
  else
    return bf16_to_f32(static_cast<const uint16_t*>(p)[e]);
}
template <bool F32>
__device__ __forceinline__ void store1(void* p, int64_t e, float v) {
  if constexpr (F32)
    static_cast<float*>(p)[e] = v;
  else
    static_cast<uint16_t*>(p)[e] = f32_to_bf16(v);
}
template <bool F32>
__device__ __forceinline__ float round_to(float v) {
  return F32 ? v : bf16_round(v);
}

// 8 values from element e on, as f32.  ANY: at any alignment.
template <bool F32, bool ANY>
__device__ __forceinline__ void load8(const void* p, int64_t e, float (&v)[8]) {
  if constexpr (F32) {
    typedef std::conditional_t<ANY, f32x4_any, f32x4_t> T;
    const T* q = reinterpret_cast<const T*>(static_cast<const float*>(p) + e);
    const f32x4_t a = q[0], b = q[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    typedef std::conditional_t<ANY, u32x4_any, u32x4_t> T;
    const u32x4_t u = *reinterpret_cast<const T*>(static_cast<const uint16_t*>(p) + e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(u[j] << 16);
      v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  }
}
template <bool F32, bool ANY>
__device__ __forceinline__ void store8(void* p, int64_t e, const float (&v)[8]) {
  if constexpr (F32) {
    typedef std::conditional_t<ANY, f32x4_any, f32x4_t> T;
    T* q = reinterpret_cast<T*>(static_cast<float*>(p) + e);
    q[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    q[1] = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    typedef std::conditional_t<ANY, u32x4_any, u32x4_t> T;
    u32x4_t u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      u[j] = (uint32_t)f32_to_bf16(v[2 * j]) | ((uint32_t)f32_to_bf16(v[2 * j + 1]) << 16);
    *reinterpret_cast<T*>(static_cast<uint16_t*>(p) + e) = u;
  }
}
// 8 bf16 weights from element j on, as they are
template <bool ANY>
__device__ __forceinline__ u32x4_t weights8(const uint16_t* w, int j) {
  return *reinterpret_cast<const std::conditional_t<ANY, u32x4_any, u32x4_t>*>(w + j);
}
// A piece of a row of d values, which is the k-th 8 of them.  ANY: a last one of fewer is the
// row's last 8, of which the first `skip` are another piece's, too: stored alike by both,
// summed by that one.
struct Piece {
  int j, skip;
};
template <bool ANY>
__device__ __forceinline__ Piece piece_at(int k, int d) {
  const int j = 8 * k, over = j + 8 - d;
  return ANY && over > 0 && over < 8 ? Piece{d - 8, over} : Piece{j, 0};
}

// The sum over a row's threads (64: a wave; 256: the workgroup), the same on all.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum_butterfly(v);
  if constexpr (TPR == 64) return v;
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // (red may hold the sum before)
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <int TPR>
__device__ __forceinline__ double row_sum(double v, double* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  if constexpr (TPR == 64) return v;
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// Codes of 4 bits show an f32's rounding: of a row's values some lie nearer to the middle of
// two codes than f32 tells apart (one in 2^18), and then the codes would go by the order of
// the sums.  So mode "mxfp8" norms in f64 and rounds once: the value goes on as f32 rounded
// to odd (the last of 24 bits set if any behind it is), which no middle of two codes is and
// no power of two that the scale goes by.
template <bool MX>
using norm_t = std::conditional_t<MX, double, float>;
__device__ __forceinline__ float to_odd(double y) {
  const uint64_t u = __builtin_bit_cast(uint64_t, y);
  const uint32_t lo = (uint32_t)u;
  const uint32_t odd = (lo & 0xe0000000u) | ((lo & 0x1fffffffu) ? 0x20000000u : 0u);
  return (float)__builtin_bit_cast(double, (u & 0xffffffff00000000ull) | odd);
}

struct NormArgs {
  const void *x, *res;
  const uint16_t* w;
  void* h;
  void* out;        // bf16 rows, or words of codes
  uint8_t* scales;  // mxfp8
  int64_t T;
  int d;
  float eps;
};

// A row by TPR threads, each C pieces of 8 values.
template <bool XF32, bool HF32, bool MX, int TPR, int C, bool ANY>
__global__ __launch_bounds__(kNT) void add_rms_norm_kernel(NormArgs a) {
  typedef norm_t<MX> sum_t;
  __shared__ sum_t red[4];
  const int lane = threadIdx.x & (TPR - 1);
  const int64_t t = (int64_t)blockIdx.x * (kNT / TPR) + (TPR == 64 ? threadIdx.x >> 6 : 0);
  if (t >= a.T) return;  // (whole rows: a wave's, or the workgroup's)
  const int64_t row = t * a.d;
  float v[C][8];
  u32x4_t wv[C];
  sum_t ss = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int j = piece_at<ANY>(lane + TPR * i, a.d).j;
    float r[8];
    if (j < a.d) {
      load8<XF32, ANY>(a.x, row + j, v[i]);
      load8<HF32, ANY>(a.res, row + j, r);
      wv[i] = weights8<ANY>(a.w, j);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[i][c] = round_to<HF32>(v[i][c] + r[c]);
    } else {
      wv[i] = u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < 8; ++c) v[i][c] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const auto [j, skip] = piece_at<ANY>(lane + TPR * i, a.d);
    if (j < a.d) store8<HF32, ANY>(a.h, row + j, v[i]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float s = c >= skip ? v[i][c] : 0.0f;
      if constexpr (MX)
        ss = __builtin_fma((double)s, (double)s, ss);
      else
        ss = __builtin_fmaf(s, s, ss);
    }
  }
  sum_t r;
  if constexpr (MX)
    r = 1.0 / sqrt(row_sum<TPR>(ss, red) / a.d + a.eps);
  else
    r = 1.0f / sqrtf(row_sum<TPR>(ss, red) / (float)a.d + a.eps);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int j = piece_at<ANY>(lane + TPR * i, a.d).j;
    float y[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float w0 = __uint_as_float(wv[i][c] << 16);
      const float w1 = __uint_as_float(wv[i][c] & 0xffff0000u);
      if constexpr (MX) {
        // (v w is exact of a bf16 row, and of an f32 one)
        y[2 * c] = to_odd((double)v[i][2 * c] * (double)w0 * r);
        y[2 * c + 1] = to_odd((double)v[i][2 * c + 1] * (double)w1 * r);
      } else {
        y[2 * c] = v[i][2 * c] * r * w0;
        y[2 * c + 1] = v[i][2 * c + 1] * r * w1;
      }
    }
    if constexpr (MX) {
      // a group is four neighbouring lanes'
      uint2 q;
      const uint32_t byte = mx8_group8(y, q);
      if (j < a.d) {
        uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + row + j);
        if constexpr (ANY)
          o[0] = q.x, o[1] = q.y;
        else
          *reinterpret_cast<uint2*>(o) = q;
        if ((lane & 3) == 0) a.scales[(row + j) >> 5] = (uint8_t)byte;
      }
    } else {
      if (j < a.d) store8<false, ANY>(a.out, row + j, y);
    }
  }
}

// Rows that no registers hold (or no piece), a workgroup each: h is written, then read back by
// the thread that wrote it.  mxfp8: 32 divides d, and a group is half a wave's.
template <bool XF32, bool HF32, bool MX>
__global__ __launch_bounds__(kNT) void add_rms_norm_any_kernel(NormArgs a) {
  typedef norm_t<MX> sum_t;
  __shared__ sum_t red[4];
  const int64_t row = (int64_t)blockIdx.x * a.d;
  sum_t ss = 0;
  for (int j = threadIdx.x; j < a.d; j += kNT) {
    const float v = round_to<HF32>(load1<XF32>(a.x, row + j) + load1<HF32>(a.res, row + j));
    store1<HF32>(a.h, row + j, v);
    if constexpr (MX)
      ss = __builtin_fma((double)v, (double)v, ss);
    else
      ss = __builtin_fmaf(v, v, ss);
  }
  sum_t r;
  if constexpr (MX)
    r = 1.0 / sqrt(row_sum<kNT>(ss, red) / a.d + a.eps);
  else
    r = 1.0f / sqrtf(row_sum<kNT>(ss, red) / (float)a.d + a.eps);
  for (int j = threadIdx.x; j < a.d; j += kNT) {
    const float h = load1<HF32>(a.h, row + j), w = bf16_to_f32(a.w[j]);
    if constexpr (MX) {
      const float y = to_odd((double)h * (double)w * r);
      uint32_t top = __float_as_uint(y) & 0x7fffffffu;
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
      const uint32_t byte = mx8_byte(top);
      static_cast<uint8_t*>(a.out)[row + j] = (uint8_t)mx8_pair(y, 0.0f, byte);
      if ((j & 31) == 0) a.scales[(row + j) >> 5] = (uint8_t)byte;
    } else {
      store1<false>(a.out, row + j, h * r * w);
    }
  }
}

struct NormVjpArgs {
  const void *dy, *h, *dh;  // dh may be null
  const uint16_t* w;
  void* dx;
  float* part;  // [gridDim.x, d]: sums of the weight's gradient
  int64_t T;
  int d;
  float eps;
};

// Rows by TPR threads each, C pieces of 8 values a thread; a thread's columns stay
// its own, so the weight's gradient adds up in registers.
template <bool YF32, bool HF32, int TPR, int C, bool ANY>
__global__ __launch_bounds__(kNT) void add_rms_norm_vjp_kernel(NormVjpArgs a) {
  constexpr int RPW = kNT / TPR;
  extern __shared__ float lds[];  // TPR == 64: the waves' weight gradients [4][d], d in eights
  const int ld = (a.d + 7) & ~7;
  __shared__ float red[8];
  const int lane = threadIdx.x & (TPR - 1), wave = threadIdx.x >> 6;
  float dw[C][8];
  u32x4_t wv[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int j = piece_at<ANY>(lane + TPR * i, a.d).j;
    wv[i] = j < a.d ? weights8<ANY>(a.w, j) : u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < 8; ++c) dw[i][c] = 0.0f;
  }
  const auto weight = [&](int i, int c) {
    const uint32_t u = wv[i][c >> 1];
    return __uint_as_float(c & 1 ? u & 0xffff0000u : u << 16);
  };
  for (int64_t t = (int64_t)blockIdx.x * RPW + (TPR == 64 ? wave : 0); t < a.T;
       t += (int64_t)gridDim.x * RPW) {
    const int64_t row = t * a.d;
    float h[C][8], dy[C][8];
    float ss = 0.0f, gh = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int j = piece_at<ANY>(lane + TPR * i, a.d).j;
      if (j < a.d) {
        load8<HF32, ANY>(a.h, row + j, h[i]);
        load8<YF32, ANY>(a.dy, row + j, dy[i]);
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) h[i][c] = dy[i][c] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int skip = piece_at<ANY>(lane + TPR * i, a.d).skip;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float s = c >= skip ? h[i][c] : 0.0f;
        ss = __builtin_fmaf(s, s, ss);
        gh = __builtin_fmaf(c >= skip ? dy[i][c] * weight(i, c) : 0.0f, s, gh);
      }
    }
    if constexpr (TPR == 64) {
      ss = wave_sum_butterfly(ss);
      gh = wave_sum_butterfly(gh);
    } else {
      ss = wave_sum_butterfly(ss);
      gh = wave_sum_butterfly(gh);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[wave] = ss, red[4 + wave] = gh;
      __syncthreads();
      ss = (red[0] + red[1]) + (red[2] + red[3]);
      gh = (red[4] + red[5]) + (red[6] + red[7]);
    }
    const float r = 1.0f / sqrtf(ss / (float)a.d + a.eps);
    const float k = r * r * (gh / (float)a.d);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int j = piece_at<ANY>(lane + TPR * i, a.d).j;
      float o[8], e[8];
      if (a.dh && j < a.d) {
        load8<HF32, ANY>(a.dh, row + j, e);
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) e[c] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        o[c] = __builtin_fmaf(r, dy[i][c] * weight(i, c) - h[i][c] * k, e[c]);
        dw[i][c] = __builtin_fmaf(dy[i][c], h[i][c] * r, dw[i][c]);
      }
      if (j < a.d) store8<HF32, ANY>(a.dx, row + j, o);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.d;
  if constexpr (TPR == 64) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const auto [j, skip] = piece_at<ANY>(lane + TPR * i, a.d);
      if (ANY && skip) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c >= skip) lds[wave * ld + j + c] = dw[i][c];
      } else if (j < a.d) {
        f32x4_t* q = reinterpret_cast<f32x4_t*>(lds + wave * ld + j);
        q[0] = f32x4_t{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
        q[1] = f32x4_t{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
      }
    }
    __syncthreads();
    for (int j = 4 * threadIdx.x; j < a.d; j += 4 * kNT) {
      const f32x4_t* q = reinterpret_cast<const f32x4_t*>(lds + j);
      const int s = ld / 4;
      const f32x4_t v = (q[0] + q[s]) + (q[2 * s] + q[3 * s]);
      if constexpr (ANY) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i < a.d) part[j + i] = v[i];
      } else {
        *reinterpret_cast<f32x4_t*>(part + j) = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const auto [j, skip] = piece_at<ANY>(lane + TPR * i, a.d);
      if (ANY && skip) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c >= skip) part[j + c] = dw[i][c];
      } else if (j < a.d) {
        store8<true, ANY>(part, j, dw[i]);
      }
    }
  }
}

// Rows that no registers hold (or no piece), in two kernels: r and r^2 c of every row, then the
// columns, a thread each, over a slice of the rows.
template <bool YF32, bool HF32>
__global__ __launch_bounds__(kNT) void norm_vjp_rows_kernel(NormVjpArgs a, float2* coef) {
  __shared__ float red[4];
  const int64_t row = (int64_t)blockIdx.x * a.d;
  float ss = 0.0f, gh = 0.0f;
  for (int j = threadIdx.x; j < a.d; j += kNT) {
    const float h = load1<HF32>(a.h, row + j);
    ss = __builtin_fmaf(h, h, ss);
    gh = __builtin_fmaf(load1<YF32>(a.dy, row + j) * bf16_to_f32(a.w[j]), h, gh);
  }
  ss = row_sum<kNT>(ss, red);
  gh = row_sum<kNT>(gh, red);
  const float r = 1.0f / sqrtf(ss / (float)a.d + a.eps);
  if (threadIdx.x == 0) coef[blockIdx.x] = make_float2(r, r * r * (gh / (float)a.d));
}
template <bool YF32, bool HF32>
__global__ __launch_bounds__(kNT) void norm_vjp_cols_kernel(NormVjpArgs a, const float2* coef,
                                                            int rows) {
  const int j = blockIdx.y * kNT + threadIdx.x;
  if (j >= a.d) return;
  const int64_t t0 = (int64_t)blockIdx.x * rows, t1 = min(t0 + rows, a.T);
  const float w = bf16_to_f32(a.w[j]);
  float dw = 0.0f;
  for (int64_t t = t0; t < t1; ++t) {
    const float2 c = coef[t];
    const float h = load1<HF32>(a.h, t * a.d + j), dy = load1<YF32>(a.dy, t * a.d + j);
    const float e = a.dh ? load1<HF32>(a.dh, t * a.d + j) : 0.0f;
    store1<HF32>(a.dx, t * a.d + j, __builtin_fmaf(c.x, dy * w - h * c.y, e));
    dw = __builtin_fmaf(dy, h * c.x, dw);
  }
  a.part[(int64_t)blockIdx.x * a.d + j] = dw;
}

// dweight [d] = the sum of part [G, d] over its rows, in f64: 32 columns
// (a line of 128 bytes) by 32 slices of the rows a workgroup.
constexpr int kJoinCols = 32, kJoinRows = 32;
__global__ __launch_bounds__(kJoinCols * kJoinRows) void norm_vjp_join_kernel(const float* part,
                                                                              int G, int d,
                                                                              float* dw) {
  __shared__ double red[kJoinRows][kJoinCols + 1];
  const int c = threadIdx.x % kJoinCols, s = threadIdx.x / kJoinCols;
  const int j = blockIdx.x * kJoinCols + c;
  double v = 0.0;
  if (j < d) {
    // 16 loads at a time (one after the other 9.6 us of 1024 rows of 2048, so 6.4; 5.0 of 512)
    int g = s;
    for (; g + 15 * kJoinRows < G; g += 16 * kJoinRows) {
      float x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = part[(int64_t)(g + k * kJoinRows) * d + j];
#pragma unroll
      for (int k = 0; k < 16; ++k) v += (double)x[k];
    }
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k)
      x[k] = g + k * kJoinRows < G ? part[(int64_t)(g + k * kJoinRows) * d + j] : 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += (double)x[k];
  }
  red[s][c] = v;
  __syncthreads();
#pragma unroll
  for (int n = kJoinRows / 2; n >= 1; n >>= 1) {
    if (s < n) red[s][c] += red[s + n][c];
    __syncthreads();
  }
  if (s == 0 && j < d) dw[j] = (float)red[0][c];
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a call's rows are split.
struct RowForm {
  bool wide;  // rows that no registers hold (or no piece): single values
  bool any;   // 16-byte accesses at any alignment, a last piece over the one before
  int tpr;   // threads per row
  int c;     // pieces of 8 a thread
};
// A wave per row holds up to kWaveMost values (the gradients fewer, with the weight's gradient
// beside them: 16384 rows of 4096 in bf16 239 us by waves, 106 by workgroups; 32768 of 2048
// 180 and 170 in f32, 127 and 125 in bf16) and needs rows enough to fill the chip; a
// workgroup per row up to 16384.
constexpr int64_t kWaveMost = 4096, kVjpWaveMost = 1024;
static_assert(kWaveMost <= 8 * 64 * 8 && kVjpWaveMost <= 8 * 64 * 2, "pieces of a wave's lanes");
RowForm row_form(int64_t T, int64_t d, bool vec, int64_t wave_most) {
  if (d > 16384 || d < 8) return {true, true, kNT, 0};
  const int tpr = d <= wave_most && T >= kNormWaveRows ? 64 : kNT;
  const int need = (int)((d + 8 * tpr - 1) / (8 * tpr));
  return {false, !vec || d % 8 != 0, tpr, need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8};
}

// CALL(threads a row, pieces a thread) by f; WIDE_WAVE(CALL, f) of a wave with more than two.
#define MLXR_NORM_FORM(CALL, f, WIDE_WAVE)          \
  do {                                              \
    if (f.tpr == 64) {                              \
      if (f.c == 1)                                 \
        CALL(64, 1);                                \
      else if (f.c == 2)                            \
        CALL(64, 2);                                \
      else                                          \
        WIDE_WAVE(CALL, f);                         \
    } else {                                        \
      switch (f.c) {                                \
        case 1: CALL(256, 1); break;                \
        case 2: CALL(256, 2); break;                \
        case 4: CALL(256, 4); break;                \
        default: CALL(256, 8);                      \
      }                                             \
    }                                               \
  } while (0)
#define MLXR_NORM_WIDE_WAVE(CALL, f) (f.c == 4 ? CALL(64, 4) : CALL(64, 8))
#define MLXR_NORM_NO_WIDE_WAVE(CALL, f) ((void)0)  // (kVjpWaveMost)

template <bool XF32, bool HF32, bool MX>
void run_norm(const NormArgs& a, const RowForm& f, hipStream_t s) {
  if (f.wide) {
    add_rms_norm_any_kernel<XF32, HF32, MX><<<(unsigned)a.T, kNT, 0, s>>>(a);
    return;
  }
  const int rpw = kNT / f.tpr;
  const unsigned grid = (unsigned)((a.T + rpw - 1) / rpw);
#define MLXR_NORM_CALL(TPR, C)                                                  \
  (f.any ? add_rms_norm_kernel<XF32, HF32, MX, TPR, C, true><<<grid, kNT, 0, s>>>(a) \
         : add_rms_norm_kernel<XF32, HF32, MX, TPR, C, false><<<grid, kNT, 0, s>>>(a))
  MLXR_NORM_FORM(MLXR_NORM_CALL, f, MLXR_NORM_WIDE_WAVE);
#undef MLXR_NORM_CALL
}

// Workgroups of the gradient's one-pass form; row slices of the other.
int vjp_groups(int64_t T, const RowForm& f) {
  if (f.wide) return (int)std::min<int64_t>((T + 63) / 64, 1024);
  const int rpw = kNT / f.tpr;
  return (int)std::min<int64_t>((T + rpw - 1) / rpw,
                                T < kNormVjpManyRows ? kNormVjpGroups : kNormVjpManyGroups);
}
struct VjpScratch {
  float* part;
  float2* coef;
};
VjpScratch carve_vjp(Carve& c, int64_t T, int64_t d) {
  const RowForm f = row_form(T, d, true, kVjpWaveMost);
  VjpScratch v;
  v.part = c.take<float>(vjp_groups(T, f) * d);
  v.coef = c.take<float2>(f.wide ? T : 0);
  return v;
}

template <bool YF32, bool HF32>
void run_norm_vjp(const NormVjpArgs& a, const RowForm& f, int G, float2* coef, hipStream_t s) {
  if (f.wide) {
    const int rows = (int)((a.T + G - 1) / G);
    norm_vjp_rows_kernel<YF32, HF32><<<(unsigned)a.T, kNT, 0, s>>>(a, coef);
    norm_vjp_cols_kernel<YF32, HF32>
        <<<dim3((unsigned)G, (unsigned)((a.d + kNT - 1) / kNT)), kNT, 0, s>>>(a, coef, rows);
    return;
  }
  const size_t lds = f.tpr == 64 ? (size_t)16 * ((a.d + 7) & ~7) : 0;
#define MLXR_NORM_CALL(TPR, C)                                                       \
  (f.any ? add_rms_norm_vjp_kernel<YF32, HF32, TPR, C, true><<<(unsigned)G, kNT, lds, s>>>(a) \
         : add_rms_norm_vjp_kernel<YF32, HF32, TPR, C, false><<<(unsigned)G, kNT, lds, s>>>(a))
  MLXR_NORM_FORM(MLXR_NORM_CALL, f, MLXR_NORM_NO_WIDE_WAVE);
#undef MLXR_NORM_CALL
}

}  // namespace

hipError_t launch_add_rms_norm(const void* x, bool x_f32, const void* residual, bool h_f32,
                               int64_t T, int64_t d, const uint16_t* w, float eps, void* h,
                               void* out, uint8_t* scales, hipStream_t s) {
  if (T == 0) return hipSuccess;
  const bool vec = aligned16(x) && aligned16(residual) && aligned16(w) && aligned16(h) &&
                   aligned16(out);
  const RowForm f = row_form(T, d, vec, kWaveMost);
  const NormArgs a{x, residual, w, h, out, scales, T, (int)d, eps};
  ProfileScope prof("add_rms_norm", s);
#define MLXR_NORM_TYPES(XF, HF) \
  (scales ? run_norm<XF, HF, true>(a, f, s) : run_norm<XF, HF, false>(a, f, s))
  if (x_f32)
    h_f32 ? MLXR_NORM_TYPES(true, true) : MLXR_NORM_TYPES(true, false);
  else
    h_f32 ? MLXR_NORM_TYPES(false, true) : MLXR_NORM_TYPES(false, false);
#undef MLXR_NORM_TYPES
  return hipGetLastError();
}

void plan_add_rms_norm_vjp(Carve& c, int64_t T, int64_t d) { (void)carve_vjp(c, T, d); }

hipError_t launch_add_rms_norm_vjp(const void* dy, bool dy_f32, const void* h, bool h_f32,
                                   int64_t T, int64_t d, const uint16_t* w, float eps,
                                   const void* dh, void* dx, float* dweight, Carve ws,
                                   hipStream_t s) {
  const VjpScratch v = carve_vjp(ws, T, d);
  const bool vec = aligned16(dy) && aligned16(h) && aligned16(w) && aligned16(dx) &&
                   aligned16(dh);
  const RowForm f = row_form(T, d, vec, kVjpWaveMost);
  const int G = T ? vjp_groups(T, f) : 0;
  const NormVjpArgs a{dy, h, dh, w, dx, v.part, T, (int)d, eps};
  ProfileScope prof("add_rms_norm_vjp", s);
  if (T) {
    if (dy_f32)
      h_f32 ? run_norm_vjp<true, true>(a, f, G, v.coef, s)
            : run_norm_vjp<true, false>(a, f, G, v.coef, s);
    else
      h_f32 ? run_norm_vjp<false, true>(a, f, G, v.coef, s)
            : run_norm_vjp<false, false>(a, f, G, v.coef, s);
  }
  norm_vjp_join_kernel<<<(unsigned)((d + kJoinCols - 1) / kJoinCols), kJoinCols * kJoinRows, 0,
                         s>>>(v.part, G, (int)d, dweight);
  return hipGetLastError();
}

}  // namespace mlxr_moe
