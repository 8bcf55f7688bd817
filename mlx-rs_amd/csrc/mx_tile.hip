// Grouped expert GEMM of microscaled 4-bit weights for many rows per expert:
// M-tiles of 32, 64 or 128 rows, the weights converted in registers.
//
// Same sums as the streaming kernel (mx_stream.hip): exact bf16 products in f32,
// in chunks of 16 inputs a matrix instruction.  A workgroup is four waves; a wave
// owns 32 gate and the same 32 up channels, or 64 down channels, for all rows of
// the tile.
//
// Weights: pieces of 8 groups (128 bytes; 4 groups under 64-row tiles) of the wave's
// 64 rows come straight to its own LDS, consecutive lanes on consecutive 16 bytes
// (loads of 32 bytes from each of 32 rows cost the address path four times the
// cycles: gate/up of c4 T=2048 212 us so, 153 with whole lines), and are then read
// to registers: lane (c, h) = (l % 32, l / 32) takes group 2 j + h of channel c in
// stage j, the operands of four v_mfma_f32_32x32x16_bf16 whose K halves are 8 inputs
// of group 2 j and 8 of group 2 j + 1.  One conversion instruction gives two
// weights, scale included: as many as there are MFMAs at 128 rows.  x is staged 64
// inputs (two groups) at a time, three stages, straight to LDS too.
// c2 T=4096: gate/up 195 us, 1.06 PFLOP/s, down 118; without any load (a copy of the
// kernel, timed) 155 and 97, where the power limit holds the matrix cores: a library
// product of 8192^3 reaches 1.46 PFLOP/s.  Without the weights' loads 172, without
// x's 192.  c4 T=2048 (40 rows an expert): gate/up 153 us for 570 MB of weights, 146 of
// them without any matrix instruction: the weights' way from memory and x's, 5 TB/s in
// all.  c2 T=64 (4 rows): gate/up 37 us, 5.7 TB/s, down 24.
#include <algorithm>
#include <type_traits>

#include "mx.hpp"
#include "prefill_reg.hpp"

namespace mlxr_moe {
namespace {

constexpr int kWaves = 4, kNT = 64 * kWaves;
typedef __attribute__((address_space(3))) void* lds_ptr;
constexpr int kXStages = 3;  // x stages of 64 inputs in LDS
// Groups of a weight piece in LDS: a 128-byte line of every row, or half of one
// under 64-row tiles, where three workgroups then fit a CU (down of c4 T=2048 102 us
// with lines and two, 96 so; c6 down T=509 39.6 and 36.5; gate/up alike).  Under
// 32-row tiles whole lines leave room for three; c6 T=100 gate/up 54 us so, 58 with
// half lines and four, 58 with two lines and two.
template <int ROWS>
constexpr int kPiece = ROWS == 64 ? 4 : 8;
template <int ROWS>
constexpr int kTileLds = kXStages * ROWS * 128 + kWaves * 2 * 512 * kPiece<ROWS>;
template <int ROWS>
constexpr int kWgs = ROWS == 128 ? 2 : 3;  // workgroups per CU
static_assert(2 * kTileLds<128> <= 160 * 1024 && 3 * kTileLds<64> <= 160 * 1024 &&
                  3 * kTileLds<32> <= 160 * 1024, "LDS");

template <int N>
__device__ __forceinline__ void wait_loads() {  // at most N loads not back
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The workgroup's barrier, when at most N of this wave's loads are not back and its
// reads of LDS are.  (__syncthreads would wait for every load to LDS.)
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A load that keeps no place in the caches.  Under 32-row tiles an expert's last tile
// (mostly its only one) reads the weights so, which nothing reads again: c2 T=64 72 us
// a pass without and 65 so, c6 down T=509 46 and 42 (46 with every tile so: an expert's
// tiles after the first then read memory again).  Whole lines only: half a line read so
// is fetched twice.  Taller tiles gain nothing (c4 T=2048 263 and 267 us).
constexpr int kNonTemporal = 2;

// The rows [slot0, slot0 + rows) of expert e against N-tile nt; last: no later tile
// has rows of e.
// NMB: 32-row blocks that hold rows.
template <bool GATED, int ROWS, int NMB>
__device__ __forceinline__ void mx_unit(const RegArgs& a, int N, int K, int e, int slot0,
                                        int rows, bool last, int nt, char* smem) {
  constexpr int TC = GATED ? 32 * kWaves : 64 * kWaves;  // channels per N-tile
  constexpr int WC = TC / kWaves;                        // ... per wave
  constexpr int kXBytes = ROWS * 128;
  constexpr int GL = kPiece<ROWS>, SPL = GL / 2;  // groups, x stages per piece
  constexpr int RPL = 64 / GL;                    // rows per load
  constexpr int kWLine = 512 * GL;                // bytes of a piece of one side
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int G = K / kMxGroup, T = K >> 6;  // groups, x stages with inputs
  const int L = (T + SPL - 1) / SPL;       // pieces
  char* xl = smem;
  char* wl = smem + kXStages * kXBytes + wave * 2 * kWLine;

  // ---- weights: pieces straight to the wave's own LDS.  Instruction i of a side
  // fills rows RPL i .. RPL i + RPL - 1, lane l the 16 bytes at position l % GL of row
  // l / GL; chunk (group) cc of row r sits at cc ^ wswz(r).  Rows past N and chunks
  // past the row are out of range: zeros.
  const uint32_t row_bytes = (uint32_t)K / 2;
  const __amdgpu_buffer_rsrc_t wr0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint32_t*>(a.w0.w) + (int64_t)e * a.e_rows * (row_bytes / 4), 0,
      (int)(N * row_bytes), kBufFlags);
  const __amdgpu_buffer_rsrc_t wr1 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint32_t*>(GATED ? a.w1.w : a.w0.w) +
          (int64_t)e * a.e_rows * (row_bytes / 4),
      0, (int)(N * row_bytes), kBufFlags);
  const int och0 = nt * TC + wave * WC;  // the wave's first channel
  const auto wswz = [&](int r) { return GL == 8 ? r & 7 : (r >> 2) & 3; };
  const int wrow = lane / GL;
  auto load_w_as = [&](int l, auto policy) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) {
        const int wch = (lane & (GL - 1)) ^ wswz(RPL * i + wrow);
        const bool ok = GL * l + wch < G;
        const int ch = och0 + (GATED ? 0 : 32 * s) + RPL * i + wrow;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            s ? wr1 : wr0, (lds_ptr)(wl + s * kWLine + 1024 * i), 16,
            ok && ch < N ? (uint32_t)ch * row_bytes + 16u * wch : kPastEnd, 16 * GL * l, 0,
            decltype(policy)::value);
      }
    }
  };
  auto load_w = [&](int l) {
    if (ROWS == 32 && last)
      load_w_as(l, std::integral_constant<int, kNonTemporal>{});
    else
      load_w_as(l, std::integral_constant<int, 0>{});
  };
  constexpr int kWLoads = GL;
  u32x4_t w[2][SPL];  // [side][stage of the piece]: the group 2 stage + h of channel c
  auto take_w = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < SPL; ++j)
        w[s][j] = *reinterpret_cast<const u32x4_t*>(wl + s * kWLine + c * 16 * GL +
                                                    16 * ((2 * j + h) ^ wswz(c)));
  };
  // ---- scales: 16 bytes of channel c (PPS pieces) at a time, by aligned words; a
  // row of an odd number of pairs starts in the middle of one
  const __amdgpu_buffer_rsrc_t sr0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.w0.scales) + (int64_t)e * a.e_rows * (G / 2), 0, N * G, kBufFlags);
  const __amdgpu_buffer_rsrc_t sr1 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(GATED ? a.w1.scales : a.w0.scales) + (int64_t)e * a.e_rows * (G / 2),
      0, N * G, kBufFlags);
  struct Scales {
    u32x4_t v;
    uint32_t past;
  };
  Scales sn[2];  // of the pieces after the current ones
  constexpr int PPS = 16 / GL;  // pieces per scale load
  auto load_sc = [&](int l) {  // pieces l .. l + PPS - 1 (l a multiple)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ch = och0 + (GATED ? 0 : 32 * s) + c;
      const uint32_t off = (uint32_t)ch * (uint32_t)G & ~3u;
      const bool ok = ch < N && GL * l < G;
      sn[s].v =
          __builtin_amdgcn_raw_buffer_load_b128(s ? sr1 : sr0, ok ? off : kPastEnd, GL * l, 0);
      sn[s].past = __builtin_amdgcn_raw_buffer_load_b32(
          s ? sr1 : sr0, ok && (G & 2) ? off + 16 : kPastEnd, GL * l, 0);
    }
  };
  uint32_t sc4[2][4];  // the pieces' scale bytes, moved so that this lane's are 0 and 2
  auto take_sc = [&](int l) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ch = och0 + (GATED ? 0 : 32 * s) + c;
      // bytes (2 i + h) of the row from group GL l on, in words of two such
      const uint32_t sh = 8 * (((uint32_t)ch * (uint32_t)G) & 3u) + 8 * h;
      const uint32_t u[5] = {sn[s].v.x, sn[s].v.y, sn[s].v.z, sn[s].v.w, sn[s].past};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = __builtin_amdgcn_alignbit(u[i + 1], u[i], sh);
        const int left = G - GL * l - 4 * i;  // zeros past the row
        sc4[s][i] = left >= 4 ? v : left > 0 ? v & 0xffffu : 0u;
      }
    }
  };

  // ---- x: straight to LDS, 64 inputs of every row a stage.  A wave's instruction j
  // fills rows 32 j + 8 wave .. + 7, lane l the 16 bytes at position l % 8 of row
  // l / 8 of them; chunk cc of row r sits at cc ^ ((r >> 1) & 7)
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.x), 0, (int)a.x_bytes, kBufFlags);
  const int xrow0 = tid >> 3, xc = (tid & 7) ^ swz(xrow0);
  load_w(0);
  load_sc(0);
  __builtin_amdgcn_sched_barrier(0);
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
  // x stage g (zeros past K) into the LDS stage at byte `at`
  auto load_x = [&](int g, int at) {
    const bool on = g < T;
#pragma unroll
    for (int j = 0; j < NMB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (lds_ptr)(xl + at + 4096 * j + 1024 * wave), 16, on ? aoff[j] : kPastEnd,
          on ? 128 * g : 0, 0, 0);
  };
#pragma unroll
  for (int g = 0; g < kXStages; ++g) load_x(g, g * kXBytes);
  // the output rows of tile rows lane and lane + 64 (the down projection)
  int orow[2] = {slot0 + min(lane, rows - 1), slot0 + min(lane + 64, rows - 1)};
  if (!GATED && a.out_by_flat) {
#pragma unroll
    for (int i = 0; i < 2; ++i) orow[i] = as_global<const int32_t>(a.sorted)[orow[i]];
  }

  f32x16_t acc[NMB][2];
#pragma unroll
  for (int i = 0; i < NMB; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  const int aswz = swz(c);
  // chunk i (16 inputs) of the x stage at byte `at`: 8 of group h of its two
  auto read_a = [&](bf16x8_t (&af)[NMB], int at, int i) {
    const char* A = xl + at + c * 128 + 16 * ((4 * h + i) ^ aswz);
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
      af[mb] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(A + 4096 * mb));
  };
  bf16x8_t af[2][NMB], bf[2];
  // side s of chunk i of stage j of the piece
  uint32_t cur[2][GL / 4];  // of the current piece
  auto pick_sc = [&](int l) {
    const int p = l & (PPS - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int k = 0; k < GL / 4; ++k) {
        cur[s][k] = sc4[s][k];
#pragma unroll
        for (int q = 1; q < PPS; ++q) cur[s][k] = p == q ? sc4[s][GL / 4 * q + k] : cur[s][k];
      }
  };
  auto weights = [&](int j, int i, int s) {
    const uint32_t v = cur[s][j >> 1];
    bf[s] = mx_weights(w[s][j][i], mx_scale((v >> (16 * (j & 1))) & 0xffu));
  };
  stage_barrier<0>();
  take_w();
  take_sc(0);
  pick_sc(0);
  read_a(af[0], 0, 0);
  weights(0, 0, 0);
  weights(0, 0, 1);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  load_w(1);
  load_sc(PPS);
  __builtin_amdgcn_sched_barrier(0);

  // ---- the pieces, SPL x stages each, four chunks of 16 inputs a stage.  The
  // operands of a chunk are read and converted during the one before it, so the
  // matrix instructions wait for neither; that is why a stage's barrier stands
  // before its last chunk, when its x has been read for good.  The x stage three
  // ahead then takes its place, and after a piece's last barrier the piece after the
  // next one the place of the next, which is in registers by then.
  // Loads are back in the order of their issue: at stage j's barrier the next
  // stage's x (two barriers old) is, when no more are out than the x stage issued
  // since, and, in the first half of a piece's stages, the weight piece issued
  // between; past the half the next piece is back too.
  int at = 0;
#pragma nounroll
  for (int l = 0; l < L; ++l) {
    const bool refill = (l & (PPS - 1)) == PPS - 1;
#pragma unroll
    for (int j = 0; j < SPL; ++j) {
      const int next = at + kXBytes < kXStages * kXBytes ? at + kXBytes : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i == 3) {
          if (j < SPL / 2)
            stage_barrier<NMB + kWLoads>();
          else
            stage_barrier<NMB>();
          load_x(SPL * l + j + kXStages, at);
          read_a(af[0], next, 0);
          if (j == SPL - 1) take_w();
        } else {
          read_a(af[(i + 1) & 1], at, i + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i == 3 && j == SPL - 1) {
          if (refill) take_sc(l + 1);
          pick_sc(l + 1);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int mb = 0; mb < NMB; ++mb)
            acc[mb][s] = mfma32x32x16(af[i & 1][mb], bf[s], acc[mb][s]);
          if (i < 3)
            weights(j, i + 1, s);
          else if (j < SPL - 1)
            weights(j + 1, 0, s);
          else
            weights(0, 0, s);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i == 3 && j == SPL - 1) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          load_w(l + 2);
          if (refill) load_sc(l + 1 + PPS);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      at = next;
    }
  }
  // nothing may be on its way to LDS when its place is used again
  wait_loads<0>();

  // ---- through the wave's own LDS, 32 rows at a time, so that every store is 16
  // bytes of a row
  uint16_t* O = reinterpret_cast<uint16_t*>(wl);
#pragma unroll
  for (int mb = 0; mb < NMB; ++mb) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 8 * (r >> 2) + 4 * h + (r & 3);
      if constexpr (GATED) {
        O[row * WC + c] = mx_bf16(mx_act(a.act, acc[mb][0][r], acc[mb][1][r]));
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) O[row * WC + 32 * s + c] = mx_bf16(acc[mb][s][r]);
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
}

template <bool GATED, int ROWS>
__global__ __launch_bounds__(kNT, kWgs<ROWS>) void mx_tile_kernel(RegLaunch L) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  RegUnit<ROWS> u;
  if (!u.place(L, blockIdx.x)) return;
  // The tile's rows end where the next tile's start (the list goes by expert, as the
  // rows do), so both records come in one step; after the last one, at the end.
  int end, next = -1;
  if (u.second) {
    u.e = 0, u.slot0 = u.tile * ROWS, end = L.rows2;
  } else {
    const int after = min(u.tile + 1, *L.a.num_tiles - 1);
    const int2 rec = *reinterpret_cast<const int2*>(L.a.tiles + 2 * u.tile);
    const int2 rec2 = *reinterpret_cast<const int2*>(L.a.tiles + 2 * after);
    const int all = L.a.offsets[L.a.E];
    u.e = __builtin_amdgcn_readfirstlane(rec.x);
    u.slot0 = __builtin_amdgcn_readfirstlane(rec.y);
    end = __builtin_amdgcn_readfirstlane(after > u.tile ? rec2.y : all);
    if (after > u.tile) next = __builtin_amdgcn_readfirstlane(rec2.x);
  }
  u.rows = min(ROWS, end - u.slot0);
  const RegArgs r = pick_reg(u.second, L.a2, L.x_bytes2, L.a, L.x_bytes);
  const bool last = u.second ? u.slot0 + ROWS >= end : next != u.e;
#define MLXR_MXU(NMB_) \
  mx_unit<GATED, ROWS, NMB_>(r, L.a.N, L.a.K, u.e, u.slot0, u.rows, last, u.nt0, smem)
  if constexpr (ROWS == 128) {
    if (u.rows > 96)
      MLXR_MXU(4);
    else if (u.rows > 64)
      MLXR_MXU(3);
    else if (u.rows > 32)
      MLXR_MXU(2);
    else
      MLXR_MXU(1);
  } else if constexpr (ROWS == 64) {
    if (u.rows > 32)
      MLXR_MXU(2);
    else
      MLXR_MXU(1);
  } else {
    MLXR_MXU(1);
  }
#undef MLXR_MXU
}

}  // namespace

hipError_t launch_mx_tile(const QGemmArgs& a, int64_t x_rows, int tile_rows, int64_t max_tiles,
                          const QGemmArgs* shared, int64_t rows2, const char* profile,
                          hipStream_t s) {
  if (tile_rows != 32 && tile_rows != 64 && tile_rows != 128) return hipErrorInvalidValue;
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
  } else if (tile_rows == 32) {
    if (a.gated)
      mx_tile_kernel<true, 32><<<grid, kNT, kTileLds<32>, s>>>(L);
    else
      mx_tile_kernel<false, 32><<<grid, kNT, kTileLds<32>, s>>>(L);
  } else {
    if (a.gated)
      mx_tile_kernel<true, 64><<<grid, kNT, kTileLds<64>, s>>>(L);
    else
      mx_tile_kernel<false, 64><<<grid, kNT, kTileLds<64>, s>>>(L);
  }
  return hipGetLastError();
}

}  // namespace mlxr_moe
