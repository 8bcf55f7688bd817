// Grouped expert GEMM of microscaled 4-bit weights for few rows per expert
// (decode).
//
//   out[p, n] = sum_k x[row(p), k] * w[e, n, k]
//
// over the work items of the dispatch (at most 8 or 16 rows of one expert), f32
// sums of exact bf16 products.  HBM-bound: 4.25 bits a weight, each read once per
// item.
//
// A workgroup is four waves: one item x 64 / KS channels.  A wave owns 16
// channels (gated: of gate and of up) over one of KS slices of the input dim;
// the slices' sums meet in LDS, added in slice order.  Per step of four groups
// (128 inputs) lane (n, q) = (l % 16, l / 16) loads the 16 bytes of channel n's
// group 4 s + q, one scale byte with it, and makes four MFMA operands of it: in
// operand i, quarter q holds inputs 8 i .. 8 i + 7 of its group, so x is read
// from LDS in the same order, and one v_mfma_f32_16x16x32_bf16 sums 8 inputs of
// four groups at once.  A lane converts 32 weights with 16 instructions and one
// scale.  D steps of loads are in flight per wave.
#include <algorithm>

#include "mx.hpp"
#include "prefill_reg.hpp"
#include "qgemm_stream.hpp"

namespace mlxr_moe {
namespace {

constexpr int kWaves = 4;

struct MxShape {
  int tiles_n;  // channel tiles per item
  int units1, items1, rows2;
};

template <bool GATED, int TT, int KS, int D>
__global__ __launch_bounds__(64 * kWaves) void mx_stream_kernel(QGemmArgs a, QGemmArgs a2,
                                                                MxShape sh) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NM = GATED ? 2 : 1;
  Unit u;
  if (!decode_unit<TT>(a, sh.tiles_n, sh.units1, sh.items1, sh.rows2, u)) return;
  const RegArgs r = pick_reg(u.shared, a2, 0, a, 0);
  const int K = a.K, G = K / kMxGroup, S = (G + 3) / 4;
  const int e = u.wk.x, row0 = u.wk.y, nt = min(u.wk.z, TT);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cw = wave / KS, kq = wave % KS;
  const int n = lane & 15, q = lane >> 4;
  const int ch = (u.tile * (kWaves / KS) + cw) * 16 + n;
  const int64_t wrow = (int64_t)e * r.e_rows + ch;
  const int SS = (S + KS - 1) / KS, s0 = kq * SS;
  const int cnt = max(min(S - s0, SS), 0);  // this wave's steps

  const u32x4_t* wp[NM];
  const uint8_t* sp[NM];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    const QWeights& W = m == 0 ? r.w0 : r.w1;
    wp[m] = reinterpret_cast<const u32x4_t*>(W.w) + wrow * G;
    sp[m] = reinterpret_cast<const uint8_t*>(W.scales) + wrow * G;
  }
  // x rows: thread k8 holds inputs 8 k8 .. 8 k8 + 7 of every row of the item
  int64_t xr[TT];
  {
    const int fl[8] = {u.fr0.x, u.fr0.y, u.fr0.z, u.fr0.w, u.fr1.x, u.fr1.y, u.fr1.z, u.fr1.w};
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int tt = min(t, nt - 1);
      if (r.x_by_slot) {
        xr[t] = row0 + tt;
      } else {
        int f;
        if constexpr (TT == 8)
          f = t < nt ? fl[t] : fl[0];
        else
          f = r.sorted[row0 + tt];
        xr[t] = r.row_map ? r.row_map[f] : f / r.row_div;
      }
    }
  }
  const int xs = 128 * S + 8;  // LDS row: 16 bytes more, so that rows start on other banks
  uint16_t* xl = reinterpret_cast<uint16_t*>(smem);
  const u32x4_t zq = {0u, 0u, 0u, 0u};
  const int per_row = 16 * S, in_row = K >> 3;
  auto load_x = [&](int k8, u32x4_t (&v)[TT]) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      v[t] = zq;
      if (t < nt && k8 < in_row)
        v[t] = *reinterpret_cast<const u32x4_t*>(r.x + xr[t] * r.x_ld + 8 * k8);
    }
  };
  auto store_x = [&](int k8, const u32x4_t (&v)[TT]) {
    if (k8 < per_row) {
#pragma unroll
      for (int t = 0; t < TT; ++t)
        if (t < nt) *reinterpret_cast<u32x4_t*>(xl + (size_t)t * xs + 8 * k8) = v[t];
    }
  };
  u32x4_t xv[TT];
  load_x(tid, xv);
  __builtin_amdgcn_sched_barrier(0);

  u32x4_t w[D][NM];
  uint32_t sc[D][NM];
  auto load_w = [&](int j, int i) {  // step i of this wave into slot j
    const int g = min(4 * (s0 + min(i, cnt - 1)) + q, G - 1);
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      w[j][m] = wp[m][g];
      sc[j][m] = sp[m][g];
    }
  };
  if (cnt > 0) {
#pragma unroll
    for (int j = 0; j < D; ++j) load_w(j, j);
  }
  __builtin_amdgcn_sched_barrier(0);
  store_x(tid, xv);
  for (int k8 = tid + 64 * kWaves; k8 < per_row; k8 += 64 * kWaves) {
    u32x4_t v[TT];
    load_x(k8, v);
    store_x(k8, v);
  }
  __syncthreads();

  f32x4_t acc[NM];
#pragma unroll
  for (int m = 0; m < NM; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // (rows past the item's read its first row: their sums go nowhere)
  const uint16_t* xa = xl + (size_t)(n < nt ? n : 0) * xs + 32 * q;
  for (int i0 = 0; i0 < cnt; i0 += D) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int i = i0 + j;
      if (i < cnt) {
        const int s = s0 + i;
        bf16x8_t xf[4];
#pragma unroll
        for (int f = 0; f < 4; ++f)
          xf[f] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(xa + 128 * s + 8 * f));
        const bool in = 4 * s + q < G;  // groups past the row: zeros (x is zero there too)
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const float scale = mx_scale(in ? sc[j][m] : 0u);
#pragma unroll
          for (int f = 0; f < 4; ++f)
            acc[m] = mfma16x16x32(xf[f], mx_weights(in ? w[j][m][f] : 0u, scale), acc[m]);
        }
      }
      load_w(j, i + D);
    }
  }

  if constexpr (KS > 1) {
    // the slices' sums, in slice order, on the first slice's wave
    f32x4_t* red = reinterpret_cast<f32x4_t*>(smem + (((size_t)TT * xs * 2 + 15) & ~size_t(15)));
#pragma unroll
    for (int m = 0; m < NM; ++m) red[(wave * NM + m) * 64 + lane] = acc[m];
    __syncthreads();
    if (kq != 0) return;
#pragma unroll
    for (int k = 1; k < KS; ++k)
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[m] += red[((wave + k) * NM + m) * 64 + lane];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * q + i;
    if (t < nt) {
      const int slot = row0 + t;
      if constexpr (GATED) {
        r.out[(int64_t)slot * r.out_ld + ch] = mx_bf16(mx_act(r.act, acc[0][i], acc[1][i]));
      } else {
        const int64_t orow =
            !r.out_by_flat ? slot : TT == 8 ? u.rec[4 + t] : r.sorted[slot];
        r.out[orow * r.out_ld + ch] = mx_bf16(acc[0][i]);
      }
    }
  }
}

}  // namespace

hipError_t launch_mx_stream(const QGemmArgs& a, int64_t max_items, const QGemmArgs* shared,
                            int64_t shared_rows, const char* profile, hipStream_t s) {
  const QGemmArgs& b = shared ? *shared : a;
  const int64_t items2 = shared ? (shared_rows + a.work_rows - 1) / a.work_rows : 0;
  const int64_t items = max_items + items2;
  const int S = (a.K / kMxGroup + 3) / 4;
  // slices: until there are 2048 waves (two per SIMD), two steps each at least
  int ks = 1;
  while (ks < kWaves && items * (a.N / 16) * ks < 2048 && S >= 4 * ks) ks *= 2;
  const int tiles_n = a.N / (16 * (kWaves / ks));
  const int nm = a.gated ? 2 : 1;
  const size_t x_lds = ((size_t)a.work_rows * (128 * S + 8) * 2 + 15) & ~size_t(15);
  const size_t lds = x_lds + (ks > 1 ? (size_t)kWaves * nm * 64 * sizeof(f32x4_t) : 0);
  const MxShape sh{tiles_n, (int)(max_items * tiles_n), (int)max_items, (int)shared_rows};
  const dim3 grid((unsigned)(items * tiles_n));
  ProfileScope prof(profile, s);
#define MLXR_MX(G_, TT_, KS_)                                                              \
  mx_stream_kernel<G_, TT_, KS_, (G_) ? 4 : 4><<<grid, 64 * kWaves, lds, s>>>(a, b, sh)
#define MLXR_MX_K(G_, TT_)   \
  do {                       \
    if (ks == 4)             \
      MLXR_MX(G_, TT_, 4);   \
    else if (ks == 2)        \
      MLXR_MX(G_, TT_, 2);   \
    else                     \
      MLXR_MX(G_, TT_, 1);   \
  } while (0)
  if (a.work_rows == kWorkRowsWide) {
    if (a.gated)
      MLXR_MX_K(true, 16);
    else
      MLXR_MX_K(false, 16);
  } else {
    if (a.gated)
      MLXR_MX_K(true, 8);
    else
      MLXR_MX_K(false, 8);
  }
#undef MLXR_MX_K
#undef MLXR_MX
  return hipGetLastError();
}

}  // namespace mlxr_moe
