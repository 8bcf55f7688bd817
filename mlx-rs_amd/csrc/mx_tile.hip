// Grouped expert GEMM of microscaled 4-bit weights for many rows per expert:
// M-tiles of 64 or 128 rows, the weights converted in registers.
//
// Same sums as the streaming kernel (mx_stream.hip): exact bf16 products in f32,
// in chunks of 16 inputs a matrix instruction.  A workgroup is four waves; a wave
// owns 32 gate and the same 32 up channels, or 64 down channels, for all rows of
// the tile.
//
// Weights: lane (c, h) = (l % 32, l / 32) loads group 2 j + h of channel c in
// load j of a 128-byte line (8 groups): 16 bytes, the operands of four
// v_mfma_f32_32x32x16_bf16 whose K halves are 8 inputs of group 2 j and 8 of
// group 2 j + 1.  One conversion instruction gives two weights, scale included,
// so the conversion is a sixth of the MFMAs' time and nothing of the weights
// passes through LDS.  x is staged 64 inputs (two groups) at a time.
#include <algorithm>

#include "mx.hpp"
#include "prefill_reg.hpp"

namespace mlxr_moe {
namespace {

constexpr int kWaves = 4, kNT = 64 * kWaves;
constexpr int kScratch = 4096;  // per wave: the epilogue's 32 rows x 64 channels
template <int ROWS>
constexpr int kTileLds = 2 * ROWS * 128 + kWaves * kScratch;

// A line of both sides: 4 loads each, and the 8 scale bytes of the line.
struct MxLine {
  u32x4_t w[2][4];
  u32x2_t sc[2];
};

// The rows [slot0, slot0 + rows) of expert e against N-tiles [nt0, nt1).
// NMB: 32-row blocks that hold rows.
template <bool GATED, int ROWS, int NMB>
__device__ __forceinline__ void mx_unit(const RegArgs& a, int N, int K, int e, int slot0,
                                        int rows, int nt0, int nt1, char* smem) {
  constexpr int TC = GATED ? 32 * kWaves : 64 * kWaves;  // channels per N-tile
  constexpr int WC = TC / kWaves;                        // ... per wave
  constexpr int kXBytes = ROWS * 128;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int G = K / kMxGroup, T = K >> 6;  // groups, x stages per tile
  const int L = (T + 3) / 4;               // lines per tile
  char* xl = smem;
  char* scratch = smem + 2 * kXBytes + wave * kScratch;

  // ---- weights and scales: the expert's rows
  const int row_bytes = K / 2;
  const __amdgpu_buffer_rsrc_t wr0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint32_t*>(a.w0.w) + (int64_t)e * a.e_rows * (row_bytes / 4), 0,
      (int)((int64_t)N * row_bytes), kBufFlags);
  const __amdgpu_buffer_rsrc_t wr1 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint32_t*>(GATED ? a.w1.w : a.w0.w) +
          (int64_t)e * a.e_rows * (row_bytes / 4),
      0, (int)((int64_t)N * row_bytes), kBufFlags);
  const gptr<const uint8_t> sp0 =
      as_global<const uint8_t>(a.w0.scales) + (int64_t)e * a.e_rows * G;
  const gptr<const uint8_t> sp1 =
      as_global<const uint8_t>(GATED ? a.w1.scales : a.w0.scales) + (int64_t)e * a.e_rows * G;
  auto channel0 = [&](int nt, int side) {
    return nt * TC + wave * WC + (GATED ? 0 : 32 * side);
  };
  int pt = nt0, pl = 0;  // the next line to load: tile, line within it
  // Every line issues the same loads; those past the row, of channels past N and
  // of lines past the unit's are out of range (zeros, no memory round trip).
  auto load_w = [&](MxLine& W) {
    const bool on = pt < nt1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ch = channel0(pt, s) + c;
      const uint32_t off = (uint32_t)ch * (uint32_t)row_bytes + 128u * pl + 16u * h;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool ok = on && ch < N && 4 * pl + j < T;
        W.w[s][j] = __builtin_amdgcn_raw_buffer_load_b128(s ? wr1 : wr0,
                                                          ok ? off + 32u * j : kPastEnd, 0, 0);
      }
      // 8 scale bytes from group 8 pl on, in one load that ends within the
      // expert's rows (shifted where that moved it); zeros past the row
      typedef uint64_t u64_a1 __attribute__((aligned(1)));
      const uint32_t so = (uint32_t)min(ch, N - 1) * (uint32_t)G + 8u * (on ? pl : 0);
      const uint32_t at = min(so, (uint32_t)N * (uint32_t)G - 8u);
      const int left = G - 8 * (on ? pl : 0);
      uint64_t v = *(gptr<const u64_a1>)((s ? sp1 : sp0) + at) >> (8 * (so - at));
      if (left < 8) v &= (1ull << (8 * left)) - 1;
      W.sc[s] = u32x2_t{(uint32_t)v, (uint32_t)(v >> 32)};
    }
    if (++pl == L) {
      pl = 0;
      ++pt;
    }
  };
  MxLine W, Wn;
  load_w(W);
  __builtin_amdgcn_sched_barrier(0);

  // ---- x: thread -> 16-byte chunk tid % 8 of the 64 inputs of rows tid / 8 +
  // 32 j; chunk cc of row r sits at cc ^ ((r >> 1) & 7)
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.x), 0, (int)a.x_bytes, kBufFlags);
  const int xrow0 = tid >> 3, xc = tid & 7;
  uint32_t aoff[NMB];
  {
    int xrow[NMB];
#pragma unroll
    for (int j = 0; j < NMB; ++j) xrow[j] = slot0 + min(xrow0 + 32 * j, rows - 1);
    if (!a.x_by_slot) {
#pragma unroll
      for (int j = 0; j < NMB; ++j) xrow[j] = as_global<const int32_t>(a.sorted)[xrow[j]];
      if (a.row_map) {
#pragma unroll
        for (int j = 0; j < NMB; ++j) xrow[j] = as_global<const int32_t>(a.row_map)[xrow[j]];
      } else {
        const float rdiv = 1.0f / (float)a.row_div;
#pragma unroll
        for (int j = 0; j < NMB; ++j) xrow[j] = div_small(xrow[j], a.row_div, rdiv);
      }
    }
#pragma unroll
    for (int j = 0; j < NMB; ++j)
      aoff[j] = xrow0 + 32 * j < rows ? (uint32_t)((int64_t)xrow[j] * a.x_ld * 2 + 16 * xc)
                                      : kPastEnd;
  }
  const int aw = xrow0 * 128 + 16 * (xc ^ swz(xrow0));
  u32x4_t xv[NMB];
  int px = 0, left_x = T * (nt1 - nt0);
  auto load_x = [&]() {
    const bool on = left_x > 0;
#pragma unroll
    for (int j = 0; j < NMB; ++j)
      xv[j] = __builtin_amdgcn_raw_buffer_load_b128(xr, on ? aoff[j] : kPastEnd,
                                                    on ? 128 * px : 0, 0);
    px = px + 1 < T ? px + 1 : 0;
    --left_x;
  };
  auto store_x = [&](int st) {
#pragma unroll
    for (int j = 0; j < NMB; ++j)
      *reinterpret_cast<u32x4_t*>(xl + st * kXBytes + aw + 4096 * j) = xv[j];
  };
  // the output rows of tile rows lane and lane + 64 (the down projection)
  int orow[2] = {slot0 + min(lane, rows - 1), slot0 + min(lane + 64, rows - 1)};
  if (!GATED && a.out_by_flat) {
#pragma unroll
    for (int i = 0; i < 2; ++i) orow[i] = as_global<const int32_t>(a.sorted)[orow[i]];
  }
  load_x();
  store_x(0);
  __syncthreads();

  f32x16_t acc[NMB][2];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < NMB; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  };
  clear();
  const int aswz = swz(c);
  auto read_a = [&](bf16x8_t (&af)[NMB], int st, int i) {
    const char* A = xl + st * kXBytes + c * 128;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
      af[mb] = as_bf16x8(
          *reinterpret_cast<const u32x4_t*>(A + 4096 * mb + 16 * ((4 * h + i) ^ aswz)));
  };

  // ---- a finished tile: through the wave's scratch, 32 rows at a time, so that
  // every store is 16 bytes of a row
  uint16_t* O = reinterpret_cast<uint16_t*>(scratch);
  auto epilogue = [&](int nt) {
    const int och0 = nt * TC + wave * WC;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      if constexpr (GATED) {
        auto rows_of = [&](auto geglu) {
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const int row = 8 * (r >> 2) + 4 * h + (r & 3);
            uint32_t v;
            if constexpr (decltype(geglu)::value)
              v = (uint32_t)geglu_bf16(bf16_round(acc[mb][0][r]), bf16_round(acc[mb][1][r])) |
                  ((uint32_t)geglu_bf16(bf16_round(acc[mb][0][r + 1]),
                                        bf16_round(acc[mb][1][r + 1]))
                   << 16);
            else
              v = swiglu_fast2(acc[mb][0][r], acc[mb][1][r], acc[mb][0][r + 1],
                               acc[mb][1][r + 1]);
            O[row * WC + c] = (uint16_t)v;
            O[(row + 1) * WC + c] = (uint16_t)(v >> 16);
          }
        };
        if (a.act == kActGeglu)
          rows_of(PfFlag<true>{});
        else
          rows_of(PfFlag<false>{});
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
          for (int s = 0; s < 2; ++s)
            O[row * WC + 32 * s + c] = __builtin_bit_cast(uint16_t, (__bf16)acc[mb][s][r]);
        }
      }
      wave_sync();
      constexpr int CPR = WC / 8;  // 16-byte runs per row
#pragma unroll
      for (int i = 0; i < 32 * CPR / 64; ++i) {
        const int id = lane + 64 * i, row = id / CPR, cc = id % CPR;
        const int trow = 32 * mb + row;
        const int64_t orw = GATED ? slot0 + trow : __shfl(orow[mb >> 1], trow & 63, 64);
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(O + row * WC + 8 * cc);
        if (trow < rows && och0 + 8 * cc < N)
          *(gptr<u32x4_t>)(as_global<uint16_t>(a.out) + orw * a.out_ld + och0 + 8 * cc) = v;
      }
      wave_sync();
    }
  };

  int xst = 0;
#pragma nounroll
  for (int nt = nt0; nt < nt1; ++nt) {
#pragma nounroll
    for (int l = 0; l < L; ++l) {
      load_w(Wn);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (4 * l + j < T) {
          load_x();
          __builtin_amdgcn_sched_barrier(0);
          float sc[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t pair = W.sc[s][j >> 1] >> (16 * (j & 1));
            sc[s] = mx_scale((h ? pair >> 8 : pair) & 0xffu);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bf16x8_t af[NMB];
            read_a(af, xst, i);
            bf16x8_t bf[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) bf[s] = mx_weights(W.w[s][j][i], sc[s]);
#pragma unroll
            for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
              for (int s = 0; s < 2; ++s) acc[mb][s] = mfma32x32x16(af[mb], bf[s], acc[mb][s]);
          }
          __builtin_amdgcn_sched_barrier(0);
          store_x(xst ^ 1);
          __syncthreads();
          xst ^= 1;
        }
      }
      W = Wn;
    }
    epilogue(nt);
    clear();
  }
}

template <bool GATED, int ROWS>
__global__ __launch_bounds__(kNT, ROWS == 128 ? 2 : 3) void mx_tile_kernel(RegLaunch L) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  RegUnit<ROWS> u;
  if (!u.place(L, blockIdx.x)) return;
  u.find_rows(L);
  const RegArgs r = pick_reg(u.second, L.a2, L.x_bytes2, L.a, L.x_bytes);
#define MLXR_MXU(NMB_) \
  mx_unit<GATED, ROWS, NMB_>(r, L.a.N, L.a.K, u.e, u.slot0, u.rows, u.nt0, u.nt1, smem)
  if constexpr (ROWS == 128) {
    if (u.rows > 96)
      MLXR_MXU(4);
    else if (u.rows > 64)
      MLXR_MXU(3);
    else if (u.rows > 32)
      MLXR_MXU(2);
    else
      MLXR_MXU(1);
  } else {
    if (u.rows > 32)
      MLXR_MXU(2);
    else
      MLXR_MXU(1);
  }
#undef MLXR_MXU
}

}  // namespace

hipError_t launch_mx_tile(const QGemmArgs& a, int64_t x_rows, int tile_rows, int64_t max_tiles,
                          const QGemmArgs* shared, int64_t rows2, const char* profile,
                          hipStream_t s) {
  if (tile_rows != 64 && tile_rows != 128) return hipErrorInvalidValue;
  const int64_t tiles2 = shared ? (rows2 + tile_rows - 1) / tile_rows : 0;
  if (max_tiles <= 0 && tiles2 <= 0) return hipSuccess;
  const QGemmArgs& b = shared ? *shared : a;
  const int cols = a.gated ? 32 * kWaves : 64 * kWaves;
  const int tiles_n = (a.N + cols - 1) / cols;
  const int units_n = tiles_n;
  const dim3 grid((unsigned)(reg_grid(max_tiles, units_n) + reg_grid(tiles2, units_n)));
  const RegLaunch L{a, tiles_n, 1, units_n, (uint32_t)(x_rows * a.x_ld * 2),
                    b, (int32_t)tiles2, (int32_t)rows2, (uint32_t)(rows2 * b.x_ld * 2)};
  ProfileScope prof(profile, s);
  if (tile_rows == 128) {
    if (a.gated)
      mx_tile_kernel<true, 128><<<grid, kNT, kTileLds<128>, s>>>(L);
    else
      mx_tile_kernel<false, 128><<<grid, kNT, kTileLds<128>, s>>>(L);
  } else {
    if (a.gated)
      mx_tile_kernel<true, 64><<<grid, kNT, kTileLds<64>, s>>>(L);
    else
      mx_tile_kernel<false, 64><<<grid, kNT, kTileLds<64>, s>>>(L);
  }
  return hipGetLastError();
}

}  // namespace mlxr_moe
