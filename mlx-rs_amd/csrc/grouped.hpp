// Products grouped by expert over rows sorted by expert: what their kernels share.
//
// Expert e has the rows offsets[e] .. offsets[e + 1] of R (offsets clamped to R); rows that no
// expert has come out as zeros.
#pragma once

#include <algorithm>

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
  int32_t chunk;   // dW: rows of a group that one tile sums over at most
  int32_t slices;  // dW: of `parts`
  int32_t max_parts, max_run;  // dW: of all groups, and of one XCD
  float* parts;    // [slices, C, J]: groups summed over in several parts
  int32_t* plan;   // dW: kPlanHead words, max_parts records, 2 words a slice.  dx: null, or
                   // dW's, to be written (with dW's chunk, slices, max_parts and max_run)
};

// dW's plan, written by one workgroup of dx or of a launch of its own: where each XCD's parts
// start (words 0 .. 8), the parts' records (expert, first row, rows, slice of a.parts or -1),
// and of every slice the expert and how many it is the first of (0: it is not the first of an
// expert's).
constexpr int kPlanHead = 16;
inline int64_t plan_words(int64_t max_parts, int64_t slices) {
  return kPlanHead + 4 * max_parts + 2 * slices;
}

// How a group's rows are cut: into n tiles of `each` rows (the last may have fewer).
struct GroupCut {
  int n, each;
};
// Forward and dx: tiles of TM rows at most, of equal numbers of blocks of 32 (16).
template <int TM>
__device__ __forceinline__ GroupCut cut_tiles(int rows) {
  const int n = (rows + TM - 1) / TM;
  constexpr int kBlock = TM < 32 ? TM : 32;
  return {n, n > 1 ? ((rows + n - 1) / n + kBlock - 1) & ~(kBlock - 1) : rows};
}
// dW: parts of `chunk` rows at most, of equal numbers of 64 rows; one for a group without
// rows, too (its dW is zeros).
__host__ __device__ __forceinline__ GroupCut cut_chunks(int rows, int chunk) {
  const int n = rows > chunk ? (rows + chunk - 1) / chunk : 1;
  return {n, n > 1 ? ((rows + n - 1) / n + 63) & ~63 : rows};
}

// A unit's place: a part of a group and a tile.
struct GroupedUnit {
  int e;            // a.E: rows that no group has
  int slot0, rows;  // the part's sorted rows
  int slice;        // dW: the slice of a.parts that it is summed in (-1: none)
  int tile;
};

__device__ __forceinline__ int clamped_offset(const GroupedArgs& a, int e) {
  return min(max(as_global<const int32_t>(a.offsets)[e], 0), (int)a.R);
}
// The inclusive results of op (of values from 0 on, 0 its neutral one) over a wave's lanes.
template <class Op>
__device__ __forceinline__ int wave_scan(int v, Op op) {
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // of the row's lanes:
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));  // one before, two,
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));  // four, eight
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // the row's before
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // the half's before
  return v;
}
struct Sum {
  __host__ __device__ int operator()(int a, int b) const { return a + b; }
};
struct Most {
  __host__ __device__ int operator()(int a, int b) const { return a > b ? a : b; }
};

// Forward and dx: the unit of a workgroup.  The groups (the rows before the first and those
// behind the last as one more each) are cut into parts of TM rows; `pick(all, u)`, of how many
// there are, gives u.tile and the part, or -1 for none.  The thread whose group has that part
// says where it is: two barriers behind the offsets (a table of all parts, searched by halves:
// one token through 8 of 256 experts 8.4 us, so 7.1).
// kFindWords words of LDS.
constexpr int kFindWords = 32;
template <int TM, class Pick>
__device__ __forceinline__ bool find_part(const GroupedArgs& a, int* lds, GroupedUnit& u,
                                          Pick pick) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int groups = a.E + 2, per = (groups + blockDim.x - 1) / blockDim.x;
  const int g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
  const auto end = [&](int g) { return g <= a.E ? clamped_offset(a, g) : (int)a.R; };
  const int first = g0 > 0 ? end(g0 - 1) : 0;
  int n = 0;
  for (int g = g0, at = first; g < g1; ++g) {
    const int to = end(g);
    n += cut_tiles<TM>(max(to - at, 0)).n;
    at = to;
  }
  const int upto = wave_scan(n, Sum{});
  if (lane == 63) lds[wave] = upto;
  __syncthreads();
  int before = upto - n, all = 0;
  for (int k = 0; k < waves; ++k) {
    const int t = lds[k];
    if (k < wave) before += t;
    all += t;
  }
  const int part = pick(__builtin_amdgcn_readfirstlane(all), u);
  if (part < 0) return false;
  if (part >= before && part < before + n) {
    int k = part - before, g = g0, at = first, to = end(g);
    GroupCut c = cut_tiles<TM>(max(to - at, 0));
    while (k >= c.n) {
      k -= c.n;
      at = to, to = end(++g);
      c = cut_tiles<TM>(max(to - at, 0));
    }
    lds[16] = g > 0 && g <= a.E ? g - 1 : a.E, lds[17] = at + k * c.each;
    lds[18] = min(to - at - k * c.each, c.each);
  }
  __syncthreads();
  u.e = __builtin_amdgcn_readfirstlane(lds[16]);
  u.slot0 = __builtin_amdgcn_readfirstlane(lds[17]);
  u.rows = __builtin_amdgcn_readfirstlane(lds[18]);
  u.slice = -1;
  return true;
}

// Upper bounds of the parts, and of the slices.
inline int64_t grouped_chunks(int64_t R, int64_t E, int64_t chunk) { return R / chunk + E; }
inline int64_t grouped_slices(int64_t R, int64_t chunk) { return R > chunk ? 2 * (R / chunk) : 0; }
// Rows that one tile of dW sums over at most: a 128th of all tiles' rows, so that a group
// that has most rows is spread over the chip, and 1024 at least.
inline int64_t grouped_chunk_rows(int64_t R, int64_t N, int64_t K) {
  const int64_t tiles = ((N + 255) / 256) * ((K + 255) / 256);
  return std::max<int64_t>(1024, (std::min(R, R * tiles / 128) + 63) / 64 * 64);
}

// dW's tiles and what its plan holds: parts, of one XCD a quarter more than an eighth, so
// that those whose parts are lighter take more of them.
constexpr int kDwTM = 128, kDwTJ = 256;
inline GroupedArgs with_plan(GroupedArgs a) {
  a.tiles_m = (a.C + kDwTM - 1) / kDwTM;
  a.tiles_j = (a.J + kDwTJ - 1) / kDwTJ;
  const int64_t parts = grouped_chunks(a.R, a.E, a.chunk);
  a.max_parts = (int32_t)parts;
  a.max_run = (int32_t)((parts + kXcds - 1) / kXcds + (parts + 31) / 32);
  return a;
}

// The threads that make a plan together: a workgroup.  (Tests make plans on the host, by one
// thread.)
struct PlanTeam {
  __device__ int tid() const { return threadIdx.x; }
  __device__ int threads() const { return blockDim.x; }
  __device__ void sync() const { __syncthreads(); }
  // op of the values of all threads before this one (0 of the first); 16 words of LDS
  template <class Op>
  __device__ int before(int v, int* words, Op op) const {
    const int lane = tid() & 63, wave = tid() >> 6;
    v = wave_scan(v, op);
    if (lane == 63) words[wave] = v;
    sync();
    v = __shfl_up(v, 1, 64);
    if (lane == 0) v = 0;
    for (int k = 0; k < wave; ++k) v = op(v, words[k]);
    return v;
  }
};

// dW: where the experts' parts lie in the order of all parts, in LDS: kGroupWords words at
// `lds`, by all of the team's threads.  Offsets that do not ascend are taken as the largest
// one up to there: of groups that lie apart there are never more parts, or slices, than the
// bounds above.
constexpr int kGroupWords = 4 * (kMaxExperts + 4) + 64;
template <class Team>
struct Groups {
  static constexpr int kStep = kMaxExperts + 4;
  const GroupedArgs& a;
  int *tab, *parts, *slices, *weights;  // offsets; parts, slices, weights before each group
  int groups;

  __host__ __device__ __forceinline__ int rows(int g) const { return tab[g + 1] - tab[g]; }
  __host__ __device__ __forceinline__ GroupCut cut(int g) const {
    return cut_chunks(rows(g), a.chunk);
  }
  // what a part costs in each of its tiles, in 32-row blocks: its own and what it costs
  // however few it has
  static __host__ __device__ __forceinline__ int weigh(GroupCut c) {
    return (c.each + 31) / 32 + 9;
  }

  __host__ __device__ __forceinline__ Groups(const GroupedArgs& a_, Team team, int* lds) : a(a_) {
    tab = lds, parts = lds + kStep, slices = lds + 2 * kStep, weights = lds + 3 * kStep;
    int* totals = lds + 4 * kStep;
    groups = a.E;
    const int tid = team.tid(), threads = team.threads();
    {
      const int per = (groups + threads) / threads;  // (of the groups + 1 offsets)
      const int e0 = Most{}(0, tid * per), e1 = e0 + per;
      int most = 0;
      for (int e = e0; e < e1 && e <= groups; ++e) {
        const int o = a.offsets[e];
        most = Most{}(most, o < a.R ? o : (int)a.R);
        tab[e] = most;
      }
      most = team.before(most, totals + 48, Most{});
      for (int e = e0; e < e1 && e <= groups; ++e) tab[e] = Most{}(tab[e], most);
      team.sync();
    }
    const int per = (groups + threads - 1) / threads;
    const int g0 = tid * per, g1 = g0 + per < groups ? g0 + per : groups;
    int n = 0, s = 0, w = 0;
    for (int g = g0; g < g1; ++g) {
      const GroupCut c = cut(g);
      n += c.n;
      if (c.n > 1) s += c.n;
      w += c.n * weigh(c);
    }
    n = team.before(n, totals, Sum{});
    s = team.before(s, totals + 16, Sum{});
    w = team.before(w, totals + 32, Sum{});
    for (int g = g0; g < g1; ++g) {
      const GroupCut c = cut(g);
      parts[g] = n, slices[g] = s, weights[g] = w;
      n += c.n;
      if (c.n > 1) s += c.n;
      w += c.n * weigh(c);
    }
    if (tid == threads - 1) parts[groups] = n, slices[groups] = s, weights[groups] = w;
    team.sync();
  }
  // The last group whose entry of t is at most v.
  __host__ __device__ __forceinline__ int search(const int* t, int v) const {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t[mid] <= v)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  }
  // The part that XCD x's start with: an eighth of all parts' weight is before it.
  __host__ __device__ __forceinline__ int start(int x) const {
    const int w = (int)((int64_t)weights[groups] * x / (int)kXcds);
    const int g = search(weights, w);
    const int p = parts[g] + (w - weights[g]) / weigh(cut(g));
    return p < parts[groups] ? p : parts[groups];
  }
};

// dW's plan, by one team (every workgroup of the products finding its part by itself
// took 80 us of 310 at 128 experts of 768 x 2048): block 0 of dx where that is asked for, too
// (a launch of its own is 4 us), else of grouped_plan_kernel.  kPlanWords words of LDS.
constexpr int kPlanWords = kGroupWords + kXcds + 1;
template <class Team>
__host__ __device__ void write_plan(const GroupedArgs& a, Team team, int* lds) {
  int* starts = lds + kGroupWords;
  const Groups<Team> groups(a, team, lds);
  const int tid = team.tid(), threads = team.threads(), cap = a.max_run;
  for (int x = tid; x <= (int)kXcds; x += threads) starts[x] = groups.start(x);
  int4* records = reinterpret_cast<int4*>(a.plan + kPlanHead);
  int2* first = reinterpret_cast<int2*>(a.plan + kPlanHead + 4 * a.max_parts);
  const int all = groups.parts[groups.groups];
  for (int p = tid; p < all; p += threads) {
    const int g = groups.search(groups.parts, p), k = p - groups.parts[g];
    const GroupCut c = groups.cut(g);
    const int left = groups.rows(g) - k * c.each;
    const int slice = c.n > 1 ? groups.slices[g] + k : -1;
    records[p] = make_int4(g, groups.tab[g] + k * c.each, left < c.each ? left : c.each, slice);
    if (slice >= 0) first[slice] = make_int2(g, k ? 0 : c.n);
  }
  team.sync();
  if (tid == 0) {
    // at most cap parts each, and few enough left for the XCDs behind
    int at = 0;
    a.plan[0] = 0;
    for (int x = 1; x <= (int)kXcds; ++x) {
      const int want = starts[x] < at + cap ? starts[x] : at + cap;
      at = Most{}(Most{}(want, all - cap * ((int)kXcds - x)), at);
      a.plan[x] = at;
    }
  }
  // (slices that no expert has)
  for (int s = groups.slices[groups.groups] + tid; s < a.slices; s += threads)
    first[s] = make_int2(0, 0);
}

// Upper bound of the parts of TM rows that find_part cuts.
inline int64_t grouped_tiles(int64_t R, int64_t E, int64_t TM) {
  return R / TM + std::min(R, E + 2);
}

// The products (grouped_tile.hip); a.tiles_m and tiles_j are the launchers' own.
// Forward: m = x, j = W [E, J, C]; dx: m = dy, j = W [E, C, J]; dW: m = dy [R, C],
// j = x, out [E, C, J].
hipError_t launch_grouped_mm(const GroupedArgs& a, hipStream_t s);
// dw: dW's arguments, whose plan dx is to write on the way, or null.  planned: it has.
hipError_t launch_grouped_dx(const GroupedArgs& a, const GroupedArgs* dw, hipStream_t s);
hipError_t launch_grouped_dw(const GroupedArgs& a, bool planned, hipStream_t s);
hipError_t launch_grouped_qmm(const GroupedArgs& a, hipStream_t s);
// grouped_mm and grouped_qmm (a.ms given) where groups have few rows (grouped_stream.hip),
// and whether they are that few.
bool grouped_streams(const GroupedArgs& a);
hipError_t launch_grouped_stream(const GroupedArgs& a, hipStream_t s);

// Rows, inputs and outputs that the kernels' grids hold: R rows by J columns.
constexpr int64_t kMaxGroupedRows = 1 << 24, kMaxGroupedDims = 1 << 16;
inline bool grouped_grid_ok(int64_t R, int64_t E, int64_t J) {
  return (grouped_tiles(R, E, 16) + 7) * ((J + 127) / 128 + 8) < ((int64_t)1 << 24);
}

}  // namespace mlxr_moe
