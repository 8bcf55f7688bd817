// The rows of each expert, for the mxfp4 tiles: a counting sort of up to
// kMxSortRows flat rows by expert in one workgroup.
//
// What the tile kernel reads of a dispatch, and no more: offsets, the sorted flat
// rows and the tile list.  Rows of an expert come in no fixed order (their ranks
// are LDS atomics): each output row's sums are the same wherever its row stands in
// a tile, so the results do not depend on it.  For gather_qmm the same launch does
// the preparation (expert and x row of each flat row).  Workgroups after the first
// clear the rows of the output that no expert takes, on CUs that the sort leaves idle.
// One launch (4072 rows 5.3 us, 20480 12.5, 32768 17.4) in place of three of 13 us
// with gaps between them, and a fourth for the preparation.
#include "common.hpp"
#include "kernels.hpp"
#include "route.hpp"

namespace mlxr_moe {
namespace {

constexpr int kThreads = 1024;
static_assert(kThreads == kMaxExperts, "a thread per expert");
constexpr int kInFlight = 8;  // ids a thread loads at a time

// Inclusive sums of two values over the workgroup's threads.
__device__ __forceinline__ void block_scan(int& a, int& b, int (*part)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int x = __shfl_up(a, m, 64), y = __shfl_up(b, m, 64);
    if (lane >= m) a += x, b += y;
  }
  if (lane == 63) part[wave][0] = a, part[wave][1] = b;
  __syncthreads();
  int x = 0, y = 0;
  for (int w = 0; w < wave; ++w) x += part[w][0], y += part[w][1];
  a += x;
  b += y;
}

__global__ __launch_bounds__(kThreads) void mx_sort_kernel(MxIds d, int tile_rows,
                                                           DispatchBuffers b, int32_t* xrow,
                                                           LeftOut left) {
  extern __shared__ uint16_t rank[];  // [n], then the sorted rows [n]
  uint16_t* const sorted = rank + d.n;
  __shared__ int count[kMaxExperts], first[kMaxExperts];
  __shared__ int part[kThreads / 64][2], bad;
  const int tid = threadIdx.x;
  const auto id_of = [&](int f) { return d.M == 1 ? d.ids[f] : d.ids[f / d.M]; };
  // whether flat row f is one to compute: its expert, and its x row, in range
  const auto good = [&](int f, int e) {
    return (uint32_t)e < (uint32_t)d.E &&
           (!d.lhs || d.lhs[f / d.M] < (uint32_t)d.x_batch);
  };
  if (blockIdx.x > 0) {
    const int wave = (int)(blockIdx.x - 1) * (kThreads / 64) + (tid >> 6);
    clear_rows<kClearRows>((int64_t)kClearRows * wave, d.n, left.y, left.N,
                           [&](int64_t f) { return good((int)f, id_of((int)f)); });
    return;
  }
  count[tid] = 0;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int f0 = tid; f0 < d.n; f0 += kInFlight * kThreads) {
    int e[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) e[i] = id_of(min(f0 + i * kThreads, d.n - 1));
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int f = f0 + i * kThreads;
      if (f >= d.n) break;
      if (good(f, e[i])) {
        rank[f] = (uint16_t)atomicAdd(&count[e[i]], 1);
      } else if (!(d.skip_minus1 && e[i] == -1)) {
        bad = 1;
      }
      if (xrow) {
        const int batch = f / d.M;
        xrow[f] = (d.lhs ? (int)d.lhs[batch] : batch / d.div) * d.M + (f - batch * d.M);
      }
    }
  }
  __syncthreads();
  const int c = count[tid];
  const int tiles = (c + tile_rows - 1) / tile_rows;
  int off = c, tile = tiles;
  block_scan(off, tile, part);
  first[tid] = off - c;
  if (tid < d.E) {
    b.offsets[tid + 1] = off;
    for (int i = 0; i < tiles; ++i) {
      b.tiles[2 * (tile - tiles + i)] = tid;
      b.tiles[2 * (tile - tiles + i) + 1] = off - c + i * tile_rows;
    }
  }
  if (tid == d.E - 1) *b.num_tiles = tile;
  if (tid == 0) {
    b.offsets[0] = 0;
    *d.status = bad;
  }
  __syncthreads();
  for (int f0 = tid; f0 < d.n; f0 += kInFlight * kThreads) {
    int e[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) e[i] = id_of(min(f0 + i * kThreads, d.n - 1));
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int f = f0 + i * kThreads;
      if (f < d.n && good(f, e[i])) sorted[first[e[i]] + rank[f]] = (uint16_t)f;
    }
  }
  __syncthreads();
  // (out of LDS in order: scattered stores of one CU took 14 of 26 us at 32768 rows)
  const int total = first[kThreads - 1] + count[kThreads - 1];
  for (int i = tid; i < total; i += kThreads) b.sorted[i] = sorted[i];
}

}  // namespace

hipError_t launch_mx_sort(const MxIds& d, int tile_rows, const DispatchBuffers& b, int32_t* xrow,
                          LeftOut left, hipStream_t s) {
  if (d.n > kMxSortRows || d.E > kMaxExperts) return hipErrorInvalidValue;
  ProfileScope prof("dispatch", s);
  static_assert(kThreads == 16 * 64, "waves of clear_groups");
  const unsigned grid = 1 + (left.y ? clear_groups(d.n) : 0);
  mx_sort_kernel<<<grid, kThreads, (size_t)d.n * 2 * sizeof(uint16_t), s>>>(d, tile_rows, b, xrow,
                                                                        left);
  return hipGetLastError();
}

}  // namespace mlxr_moe
