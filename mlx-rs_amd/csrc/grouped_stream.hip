// Products grouped by expert where the groups have few rows: the forward product
//   y[r, n] = sum_k x[r, k] W[e(r)][n, k]
// in bf16, and of e4m3 rows by e2m1 weights with a power-of-two scale per 32.
//
// A group's rows, up to 16 of them, are one operand of a 16 x 16 matrix instruction, 16
// rows of W the other; both go straight from memory to the lanes that the instruction wants
// them in (16 bytes each), as W's rows are used once.  Bound by HBM, and in the smallest
// calls by the latency from the offsets to the last load: a wave asks for all of its chunk
// before it waits.  The inputs of a row are split over `ksplit` of a workgroup's eight
// waves, whose sums are joined in LDS in order.
//
// Measured: one token's 8 experts of 512 x 2048 7 us (3.5 at a copy's rate), in 8 by 4 bits 8
// of 768 x 2048 7 us; 640 rows of 512 experts of 2048 x 512 in 8 by 4 bits 50 us, floor 43.
#include <algorithm>

#include "grouped.hpp"

namespace mlxr_moe {
namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kRows = 16, kWaves = 8;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t stream_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(
      const_cast<void*>(p), 0, (int)(uint32_t)min(max(bytes, (int64_t)0), (int64_t)0xFFFFF000),
      kBufFlags);
}

// F8: of 8-bit rows by 4-bit weights.  A wave's column tile is 16 columns; a workgroup takes
// `per` of its tiles of kWaves / ksplit of them.
template <bool F8>
__global__ __launch_bounds__(64 * kWaves) void grouped_stream_kernel(GroupedArgs a, int ksplit,
                                                                     int per) {
  constexpr int STEP = F8 ? 128 : 32;  // inputs of an instruction
  constexpr int CH = F8 ? 2 : 4;       // steps of a chunk
  constexpr int XL = F8 ? 2 : 1;       // loads of x a step
  __shared__ union {
    int words[kFindWords];
    f32x4_t sums[2][kWaves][64];
  } lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int csplit = kWaves / ksplit, kk = wave / csplit;
  // ---- the workgroup's unit: a part and `per` column tiles.  XCDs take runs of them (a
  // part's, one part after the other): an expert of several parts is read by one of them.
  const int runs = (a.tiles_j + per - 1) / per;
  GroupedUnit u;
  const bool found = find_part<kRows>(a, lds.words, u, [&](int parts, auto& v) {
    const int x = blockIdx.x % kXcds, i = blockIdx.x / kXcds;
    const int64_t all = (int64_t)parts * runs, at = all * x / kXcds + i;
    const int part = (int)(at / runs);
    v.tile = (int)(at - (int64_t)part * runs) * per;
    return at < all * (x + 1) / kXcds ? part : -1;
  });
  if (!found) return;
  __syncthreads();  // (the sums take the words' place)
  const int e = u.e, slot0 = u.slot0, rows = u.rows;
  const int tile0 = __builtin_amdgcn_readfirstlane(u.tile);
  const int tiles = min(per, a.tiles_j - tile0);
  const int wcol0 = (tile0 * csplit + wave % csplit) * 16;  // the wave's columns: of tile t
  const int es = a.out_f32 ? 4 : 2;                         // from 16 csplit t on
  uint32_t xrow = c;    // the lane's row of x
  bool xok = c < rows;  // (false, too, of an index that names none)
  // lane: of row c columns 4 g .. + 3 of a tile; zeros where no row of x is, whatever W holds
  const auto put = [&](int t, f32x4_t v) {
    const int col = wcol0 + 16 * csplit * t + 4 * g;
    if (c >= rows || col >= a.J) return;
    if (!xok) v = f32x4_t{0, 0, 0, 0};
    char* p = static_cast<char*>(a.out) + ((int64_t)(slot0 + c) * a.J + col) * es;
    if (a.out_f32)
      *reinterpret_cast<f32x4_t*>(p) = v;
    else
      *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  };
  if (e == a.E) {  // rows that no group has
    if (kk == 0)
      for (int t = 0; t < tiles; ++t) put(t, f32x4_t{0, 0, 0, 0});
    return;
  }

  // ---- where the operands are
  const int G = a.C / 32;
  const int64_t ldx = F8 ? (int64_t)a.C : (int64_t)a.C * 2, ldw = F8 ? a.C / 2 : (int64_t)a.C * 2;
  const bool mapped = a.rows != nullptr;
  const int64_t w0 = (int64_t)e * a.J + wcol0, wrows = a.J - wcol0;
  const __amdgpu_buffer_rsrc_t wr =
      stream_rsrc(static_cast<const char*>(a.j) + w0 * ldw, wrows * ldw);
  const __amdgpu_buffer_rsrc_t wsr = stream_rsrc(a.js + w0 * G, F8 ? wrows * G : 0);
  const __amdgpu_buffer_rsrc_t xr =
      stream_rsrc(static_cast<const char*>(a.m) + (mapped ? 0 : slot0 * ldx),
                  (mapped ? a.x_rows : rows) * ldx);
  const __amdgpu_buffer_rsrc_t xsr =
      stream_rsrc(a.ms + (mapped ? 0 : (int64_t)slot0 * G),
                  F8 ? (mapped ? a.x_rows : rows) * (int64_t)G : 0);
  const int steps = (a.C + STEP - 1) / STEP;
  const int s0 = steps * kk / ksplit, s1 = steps * (kk + 1) / ksplit;
  const int chunks = ((steps + ksplit - 1) / ksplit + CH - 1) / CH;  // (of all waves as many)

  struct Chunk {
    u32x4_t w[CH], x[CH][XL];
    uint32_t ws[CH], xs[CH];
  };
  // the first of this lane's inputs of W in step s
  const auto at = [&](int s) { return STEP * s + (STEP / 4) * g; };
  const auto load_w = [&](Chunk& k, int t, int s) {
    const uint32_t r = 16 * csplit * t + c;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const bool ok = s + i < s1 && at(s + i) < a.C;
      const uint32_t off = r * (uint32_t)ldw + (F8 ? at(s + i) / 2 : 2 * at(s + i));
      k.w[i] = __builtin_amdgcn_raw_buffer_load_b128(wr, ok ? off : kPastEnd, 0, 0);
      if constexpr (F8)
        k.ws[i] = __builtin_amdgcn_raw_buffer_load_b8(
            wsr, ok ? r * G + at(s + i) / 32 : kPastEnd, 0, 0);
    }
  };
  const auto load_x = [&](Chunk& k, int s) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int l = 0; l < XL; ++l) {
        // (F8: 16 inputs of each of the step's halves)
        const int j = F8 ? STEP * (s + i) + 64 * l + 16 * g : at(s + i);
        const bool ok = xok && s + i < s1 && j < a.C;
        const uint32_t off = xrow * (uint32_t)ldx + (F8 ? j : 2 * j);
        k.x[i][l] = __builtin_amdgcn_raw_buffer_load_b128(xr, ok ? off : kPastEnd, 0, 0);
      }
      if constexpr (F8)
        k.xs[i] = __builtin_amdgcn_raw_buffer_load_b8(
            xsr, xok && s + i < s1 && at(s + i) < a.C ? xrow * G + at(s + i) / 32 : kPastEnd, 0, 0);
    }
  };
  f32x4_t acc = {0, 0, 0, 0};
  const auto multiply = [&](const Chunk& k) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const u32x4_t w = k.w[i];
      if constexpr (F8) {
        const i32x8_t wf{(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
        const u32x4_t l = k.x[i][0], h = k.x[i][XL - 1];
        const i32x8_t xf{(int)l.x, (int)l.y, (int)l.z, (int)l.w,
                         (int)h.x, (int)h.y, (int)h.z, (int)h.w};
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc, 4, 0, 0, k.ws[i], 0,
                                                               k.xs[i]);
      } else {
        acc = mfma16x16x32(as_bf16x8(w), as_bf16x8(k.x[i][0]), acc);
      }
    }
  };
  // ---- all tiles' chunks, one behind the other; the one ahead on its way
  Chunk set[2];
  int lt = 0, ls = 0;  // of the next to load: its tile, its chunk
  const auto load = [&](Chunk& k) {
    if (lt < tiles) {
      load_w(k, lt, s0 + ls * CH);
      load_x(k, s0 + ls * CH);
    }
    if (++ls == chunks) ls = 0, ++lt;
  };
  load_w(set[0], 0, s0);  // (these do not wait for the rows' indices)
  if (mapped && xok) {
    const int x = as_global<const int32_t>(a.rows)[slot0 + c];
    xok = x >= 0 && x < a.x_rows;
    xrow = (uint32_t)x;
  }
  load_x(set[0], s0);
  if (++ls == chunks) ls = 0, ++lt;
  int ct = 0, cs = 0;  // of the next to multiply
  const auto step = [&](Chunk& now, Chunk& next) {
    load(next);
    __builtin_amdgcn_sched_barrier(0);
    multiply(now);
    if (++cs < chunks) return;
    cs = 0;
    if (ksplit == 1) {
      put(ct, acc);
    } else {
      lds.sums[ct & 1][wave][lane] = acc;
      __syncthreads();  // (the place before it was read before the last one)
      if (kk == 0) {
        f32x4_t v = acc;
        for (int k = 1; k < ksplit; ++k) v += lds.sums[ct & 1][k * csplit + wave][lane];
        put(ct, v);
      }
    }
    acc = f32x4_t{0, 0, 0, 0};
    ++ct;
  };
#pragma nounroll
  while (ct < tiles) {
    step(set[0], set[1]);
    if (ct >= tiles) break;
    step(set[1], set[0]);
  }
}

// A wave's work is about 1024 inputs of 16 columns (32 KB of bf16 weights), 2048 of the 8-
// and 4-bit kind (16 KB), of one column tile or several: more leaves the last workgroups
// alone, less pays for finding the unit.  128 rows of 256 experts, J 512, C 2048: 41 us; all
// 2048 inputs in one wave 54, 512 of them 44.  8 by 4 bits, 640 rows of 512 experts, J 2048,
// C 512: four tiles 54 us, two 69, one 93.  Units too few to fill the chip are split further,
// down to 256 inputs a wave: 8 rows of those 256 experts 8.9 us, at 1024 inputs 14.7.
template <bool F8>
hipError_t stream(GroupedArgs a, hipStream_t s) {
  const int target = F8 ? 2048 : 1024;
  const int64_t parts = grouped_tiles(a.R, a.E, kRows);
  int ksplit = 1, per = std::max(1, target / a.C);
  while (ksplit < kWaves && a.C / ksplit > target) ksplit *= 2;
  int64_t runs;
  for (;;) {
    const int cols = kWaves / ksplit * 16;
    a.tiles_j = (a.J + cols - 1) / cols;
    per = std::min(per, a.tiles_j);
    runs = (a.tiles_j + per - 1) / per;
    if (parts * runs >= 512) break;
    if (per > 1)
      per /= 2;
    else if (ksplit < kWaves && a.C / ksplit >= 512)
      ksplit *= 2;
    else
      break;
  }
  const int64_t grid = (parts * runs + kXcds - 1) / kXcds * kXcds;
  if (grid * 64 * kWaves > UINT32_MAX) return hipErrorInvalidValue;  // (the callers check)
  grouped_stream_kernel<F8><<<(unsigned)grid, 64 * kWaves, 0, s>>>(a, ksplit, per);
  return hipGetLastError();
}

}  // namespace

// Against the tiles (grouped_tile.hip, 64 x 128 of these calls): where the tiles leave half
// of the chip alone, up to 8 rows a group (8 experts of 768 x 2048: 2 rows 7.7 us against
// 17.2, 32 11.5 against 17.8, but 128 18.8 against 18.6; 8 by 4 bits 6.7 against 12.8, 8.8
// against 12.9, 14.1 against 14.4).  Else up to 2 rows a group in bf16 (256 experts of 512 x
// 2048: 512 rows 75 us against 91, 2048 rows 124 against 121), and 8 by 4 bits up to 4 of at
// most 512 inputs, where the tiles' loop is over before it is filled (512 experts of 2048 x
// 512: 640 rows 54 against 79, 2560 97 against 108, 5120 135 against 121; but 256 of 512 x
// 2048, 128 rows 25 against 17).
bool grouped_streams(const GroupedArgs& a) {
  const bool few = grouped_tiles(a.R, a.E, 64) * ((a.J + 127) / 128) < 256;
  if (few) return a.R <= 8 * (int64_t)a.E;
  return a.ms ? a.C <= 512 && a.R <= 4 * (int64_t)a.E : a.R <= 2 * (int64_t)a.E;
}
hipError_t launch_grouped_stream(const GroupedArgs& a, hipStream_t s) {
  return a.ms ? stream<true>(a, s) : stream<false>(a, s);
}

}  // namespace mlxr_moe
