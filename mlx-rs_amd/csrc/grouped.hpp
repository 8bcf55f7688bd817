// Products grouped by expert over rows sorted by expert: what their kernels share.
//
// Expert e has the rows offsets[e] .. offsets[e + 1] of R (offsets clamped to R).
#pragma once

#include "common.hpp"
#include "kernels.hpp"
#include "mx.hpp"
#include "prefill_reg.hpp"

namespace mlxr_moe {

typedef __attribute__((address_space(3))) char* lds_ptr;

struct GroupedArgs {
  const void* m;       // rows of the output: x, or dy; of dW: dy
  const void* j;       // columns of the output: W; of dW: x
  const uint8_t* ms;   // scale bytes of x (mxfp8) ...
  const uint8_t* js;   // ... and of W (mxfp4)
  const int32_t* offsets;
  const int32_t* rows;  // the row of x of each sorted row (null: the row itself)
  void* out;
  int64_t R;       // sorted rows
  int64_t x_rows;  // rows of x
  int32_t E;
  int32_t J;        // output columns
  int32_t C;        // inputs summed over (dW: the output's rows)
  int32_t tiles_j;  // column tiles
  int32_t tiles_m;  // row tiles of one expert (dW)
  int32_t out_f32;
};

// A tile's group and rows.
struct GroupedTile {
  int e;  // E: rows that no group has
  int64_t slot0, rows;
};

__device__ __forceinline__ int64_t group_at(const GroupedArgs& a, int e) {
  return min(max((int64_t)a.offsets[e], (int64_t)0), a.R);
}

// Workgroup b's unit of those that the groups' tiles of TM rows make with tiles_j
// column tiles each, the rows behind the last group (expert E) among them.  Every wave
// does this by itself: lane l counts the tiles of a run of groups, a scan over the
// lanes places them.  Units go to the XCDs in runs, so that one L2 sees an expert's.
// False: no such unit.
template <int TM>
__device__ __forceinline__ bool find_tile(const GroupedArgs& a, int b, GroupedTile& t, int& tj) {
  const int lane = threadIdx.x & 63;
  const int per = (a.E + 64) / 64;  // groups a lane, of E + 1
  const int g0 = lane * per, g1 = min(g0 + per, a.E + 1);
  int count = 0;
  if (g0 < g1) {
    int64_t at = group_at(a, g0);
    for (int g = g0; g < g1; ++g) {
      const int64_t end = g < a.E ? group_at(a, g + 1) : a.R;
      if (end > at) count += (int)((end - at + TM - 1) / TM);
      at = end;
    }
  }
  int incl = count;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int v = __shfl_up(incl, s, 64);
    if (lane >= s) incl += v;
  }
  const int total = __builtin_amdgcn_readlane(incl, 63);
  const int units = total * a.tiles_j;
  const int per_x = (units + (int)kXcds - 1) / (int)kXcds;
  const int u = (b % (int)kXcds) * per_x + b / (int)kXcds;
  if (b / (int)kXcds >= per_x || u >= units) return false;
  const int tile = u / a.tiles_j;
  tj = u - tile * a.tiles_j;
  const uint64_t mine = __ballot(incl > tile);
  const int owner = __builtin_ctzll(mine);
  int e = 0, part = 0;
  if (lane == owner) {
    int left = tile - (incl - count);
    int64_t at = group_at(a, g0);
    for (int g = g0; g < g1; ++g) {
      const int64_t end = g < a.E ? group_at(a, g + 1) : a.R;
      const int n = end > at ? (int)((end - at + TM - 1) / TM) : 0;
      if (left < n) {
        e = g, part = left;
        break;
      }
      left -= n;
      at = end;
    }
  }
  e = __builtin_amdgcn_readlane(e, owner);
  part = __builtin_amdgcn_readlane(part, owner);
  const int64_t at = group_at(a, e), end = e < a.E ? group_at(a, e + 1) : a.R;
  t.e = e;
  t.slot0 = at + (int64_t)part * TM;
  t.rows = min(end - t.slot0, (int64_t)TM);
  return true;
}

// Upper bound of the tiles of TM rows (find_tile's total).
inline int64_t grouped_tiles(int64_t R, int64_t E, int64_t TM) {
  return R / TM + (R < E + 1 ? R : E + 1);
}

// The products (grouped_tile.hip); a.tiles_m and tiles_j are the launchers' own.
// Forward: m = x, j = W [E, J, C]; dx: m = dy, j = W [E, C, J]; dW: m = dy [R, C],
// j = x, out [E, C, J].
hipError_t launch_grouped_mm(const GroupedArgs& a, hipStream_t s);
hipError_t launch_grouped_dx(const GroupedArgs& a, hipStream_t s);
hipError_t launch_grouped_dw(const GroupedArgs& a, hipStream_t s);
hipError_t launch_grouped_qmm(const GroupedArgs& a, hipStream_t s);

// Rows, inputs and outputs that the kernels' grids hold: R rows by J columns.
constexpr int64_t kMaxGroupedRows = 1 << 24, kMaxGroupedDims = 1 << 16;
inline bool grouped_grid_ok(int64_t R, int64_t E, int64_t J) {
  return (grouped_tiles(R, E, 16) + 8) * ((J + 127) / 128 + 8) < ((int64_t)1 << 24);
}

}  // namespace mlxr_moe
