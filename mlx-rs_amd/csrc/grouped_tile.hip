// Products grouped by expert over ragged groups of rows, in tiles on the matrix cores:
//   forward   y[r, n]     = sum_k x[r, k] W[e(r)][n, k]
//   dx        dx[r, k]    = sum_n dy[r, n] W[e(r)][n, k]
//   dW        dW[e][n, k] = sum_{r of e} dy[r, n] x[r, k]
// in bf16 with f32 sums, and the forward product of e4m3 rows by e2m1 weights, each
// with a power-of-two scale per 32 (modes mxfp8 and mxfp4).
//
// One kernel body.  An output tile is TM x TJ; a stage of 64 inputs (128 of the 8- and
// 4-bit ones) of both operands goes straight to LDS by 16-byte loads while the stage
// before is multiplied.  An operand whose inputs run along memory (x and W forward, dy
// of dx) lies in LDS as 128-byte rows; one whose inputs run across rows (W of dx, both
// of dW) as rows of columns, read transposed by ds_read_b64_tr_b16.
#include <algorithm>

#include "grouped.hpp"
#include "nn.hpp"

namespace mlxr_moe {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

enum { kForward, kDx, kDw, kForward8 };

template <int KIND>
constexpr bool kMTrans = KIND == kDw;
template <int KIND>
constexpr bool kJTrans = KIND == kDw || KIND == kDx;

// Bytes of a stage.  8-bit: TJ rows of 64 bytes of weights.
template <int KIND, int TM, int TJ>
constexpr int kStage = TM * 128 + TJ * (KIND == kForward8 ? 64 : 128);
// ... and of the scales of four stages: 16 bytes a row
template <int KIND, int TM, int TJ>
constexpr int kScales = KIND == kForward8 ? 16 * (TM + TJ) : 0;
template <int KIND, int TM, int TJ, int STAGES>
constexpr int kTileLds = STAGES * kStage<KIND, TM, TJ> + 2 * kScales<KIND, TM, TJ>;

// Where 32-byte piece p of row r of a transposed operand lies: at p ^ tkey(r).  The four
// rows and the two neighbouring pieces that half a wave reads at once lie in eight
// different eighths of 256 bytes so.
__device__ __forceinline__ int tkey(int r) { return (r & 3) | ((r & 1) << 2); }

// One load of 16 bytes a lane to consecutive LDS
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, char* to, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)to, 16, off, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0,
                                           (int)(uint32_t)min(max(bytes, (int64_t)0),
                                                              (int64_t)0xFFFFF000),
                                           kBufFlags);
}

// The tile of output rows [row0, row0 + rows) and columns [col0, ..): rows of the group
// (forward, dx) or of dW.  slot0, len: the group's first row and rows (dW).
template <int KIND, int TM, int TJ, int WM, int WJ, int STAGES, int NMB>
__device__ __forceinline__ void tile_unit(const GroupedArgs& a, int e, int64_t slot0, int64_t len,
                                          int row0, int rows, int col0, char* smem) {
  constexpr bool F8 = KIND == kForward8, MT = kMTrans<KIND>, JT = kJTrans<KIND>;
  constexpr int NW = WM * WJ;
  constexpr int MB = TM / WM / 32, NB = TJ / WJ / 32;  // 32 x 32 blocks of a wave
  constexpr int NA = NMB > 0 ? NMB : 1;
  constexpr int kM = TM * 128;  // the J operand's place in a stage
  constexpr int ML = TM / 8 / NW, JL = (F8 ? TJ / 16 : TJ / 8) / NW;  // loads a wave
  static_assert(ML >= 1 && JL >= 1 && MB >= 1 && NB >= 1, "tile");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WJ, wj = wave % WJ;
  const int c = lane & 31, h = lane >> 5;

  // ---- where the operands start, how far apart their rows are, how many stages
  const int esM = F8 ? 1 : 2;
  const int64_t ldm = MT ? (int64_t)a.C * 2 : (int64_t)a.C * esM;  // bytes
  const int64_t ldj = JT ? (int64_t)a.J * 2 : F8 ? (int64_t)a.C / 2 : (int64_t)a.C * 2;
  const bool mapped = a.rows != nullptr;  // x's rows (M forward, J of dW)
  const int64_t cn = MT ? len : a.C;      // inputs
  constexpr int SI = F8 ? 128 : 64;       // a stage's
  const int T = (int)((cn + SI - 1) / SI);

  // ---- M
  const char* mp;
  int64_t mbytes;
  uint32_t moff[ML];
  if constexpr (MT) {
    mp = static_cast<const char*>(a.m) + slot0 * ldm + 2 * (int64_t)row0;
    mbytes = len * ldm - 2 * (int64_t)row0;
    constexpr int P = TM / 8;  // 16-byte pieces a row
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      const int r = (wave * ML + i) * (64 / P) + lane / P, p = lane % P;
      moff[i] = (uint32_t)(r * ldm) + 32 * ((p >> 1) ^ tkey(r)) + 16 * (p & 1);
    }
  } else {
    const bool map = mapped && KIND != kDx;
    mp = static_cast<const char*>(a.m) + (map ? 0 : (slot0 + row0) * ldm);
    mbytes = map ? a.x_rows * ldm : rows * ldm;
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      const int r = (wave * ML + i) * 8 + (lane >> 3);
      int64_t at = (int64_t)r * ldm;
      bool ok = r < rows;
      if (map) {
        const int x = as_global<const int32_t>(a.rows)[slot0 + row0 + min(r, rows - 1)];
        ok = ok && x >= 0 && x < a.x_rows;
        at = x * ldm;
      }
      moff[i] = ok ? (uint32_t)at + 16 * ((lane & 7) ^ swz(r)) : kPastEnd;
    }
  }
  // ---- J
  const char* jp;
  int64_t jbytes;
  uint32_t joff[JL];
  if constexpr (JT) {
    const bool map = KIND == kDw && mapped;
    jp = static_cast<const char*>(a.j) + 2 * (int64_t)col0 +
         (KIND == kDw ? (map ? 0 : slot0 * ldj) : (int64_t)e * a.C * ldj);
    jbytes = (KIND == kDw ? (map ? a.x_rows : len) : (int64_t)a.C) * ldj - 2 * (int64_t)col0;
    constexpr int P = TJ / 8;
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      const int r = (wave * JL + i) * (64 / P) + lane / P, p = lane % P;
      joff[i] = (map ? 0u : (uint32_t)(r * ldj)) + 32 * ((p >> 1) ^ tkey(r)) + 16 * (p & 1);
    }
  } else {
    jp = static_cast<const char*>(a.j) + ((int64_t)e * a.J + col0) * ldj;
    jbytes = (int64_t)(a.J - col0) * ldj;
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      const int r = F8 ? (wave * JL + i) * 16 + (lane >> 2) : (wave * JL + i) * 8 + (lane >> 3);
      const int p = F8 ? (lane & 3) ^ ((r >> 2) & 3) : (lane & 7) ^ swz(r);
      joff[i] = (uint32_t)(r * ldj) + 16 * p;
    }
  }
  // the rows of x of a stage of dW, found a stage ahead
  int xrow[KIND == kDw ? JL : 1];
  auto find_x = [&](int t) {
    if constexpr (KIND == kDw) {
      if (mapped) {
        constexpr int P = TJ / 8;
#pragma unroll
        for (int i = 0; i < JL; ++i) {
          const int64_t r = (int64_t)t * 64 + (wave * JL + i) * (64 / P) + lane / P;
          xrow[i] = r < len ? as_global<const int32_t>(a.rows)[slot0 + r] : -1;
        }
      }
    }
  };

  // ---- a stage's loads
  const int mchunks = F8 ? a.C / 16 : a.C / 8;  // 16-byte pieces of an M row, of a J row
  const int jchunks = F8 ? a.C / 32 : a.C / 8;
  auto issue = [&](int t, char* S) {
    const int64_t mo = MT ? (int64_t)t * 64 * ldm : (int64_t)t * 128;
    const __amdgpu_buffer_rsrc_t mr = rsrc(mp + mo, mbytes - mo);
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      bool ok = true;
      if constexpr (!MT)
        ok = 8 * t + ((lane & 7) ^ swz((wave * ML + i) * 8 + (lane >> 3))) < mchunks;
      load_lds(mr, S + (wave * ML + i) * 1024, ok ? moff[i] : kPastEnd);
    }
    if constexpr (KIND == kDw) {
      if (mapped) {
        const __amdgpu_buffer_rsrc_t jr = rsrc(jp, jbytes);
#pragma unroll
        for (int i = 0; i < JL; ++i)
          load_lds(jr, S + kM + (wave * JL + i) * 1024,
                   xrow[i] >= 0 && xrow[i] < a.x_rows ? joff[i] + (uint32_t)(xrow[i] * ldj)
                                                      : kPastEnd);
        return;
      }
    }
    const int64_t jo = JT ? (int64_t)t * 64 * ldj : (int64_t)t * (F8 ? 64 : 128);
    const __amdgpu_buffer_rsrc_t jr = rsrc(jp + jo, jbytes - jo);
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      bool ok = true;
      if constexpr (!JT) {
        const int r = F8 ? (wave * JL + i) * 16 + (lane >> 2) : (wave * JL + i) * 8 + (lane >> 3);
        const int p = F8 ? (lane & 3) ^ ((r >> 2) & 3) : (lane & 7) ^ swz(r);
        ok = (F8 ? 4 : 8) * t + p < jchunks;
      }
      load_lds(jr, S + kM + (wave * JL + i) * 1024, ok ? joff[i] : kPastEnd);
    }
  };
  // ---- the scales of stages 4 q .. 4 q + 3, 16 bytes a row (zeros past the row's)
  const int G = a.C / 32;
  char* scl = smem + STAGES * kStage<KIND, TM, TJ>;
  auto issue_scales = [&](int q, char* S) {
    if constexpr (F8) {
      for (int r = tid; r < TM + TJ; r += 64 * NW) {
        const bool isj = r >= TM;
        const int rr = isj ? r - TM : r;
        const uint8_t* p = nullptr;
        if (isj) {
          if (col0 + rr < a.J) p = a.js + ((int64_t)e * a.J + col0 + rr) * G;
        } else if (rr < rows) {
          int64_t x = slot0 + row0 + rr;
          if (mapped) {
            x = as_global<const int32_t>(a.rows)[x];
            if (x < 0 || x >= a.x_rows) x = -1;
          }
          if (x >= 0) p = a.ms + x * G;
        }
        uint32_t v[4] = {0, 0, 0, 0};
        if (p) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (16 * q + i < G) v[i >> 2] |= (uint32_t)p[16 * q + i] << (8 * (i & 3));
        }
        *reinterpret_cast<u32x4_t*>(S + 16 * r) = u32x4_t{v[0], v[1], v[2], v[3]};
      }
    }
  };

  // ---- the products of a stage
  f32x16_t acc[NA][NB];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  const int m0 = wm * MB, j0 = wj * NB;  // the wave's first blocks
  // transposed: byte of the lane's four values of block 0, rows 8 h + (lane % 16) / 4
  const int ti = lane & 15, tg = (lane >> 4) & 1;
  const int tlow = ((tg ^ tkey(ti >> 2)) << 5) + 8 * (ti & 3);
  auto frag = [&](const char* O, int blk, int ks, bool trans, int row_bytes) -> bf16x8_t {
    if (!trans)
      return as_bf16x8(*reinterpret_cast<const u32x4_t*>(O + blk * 4096 + c * 128 +
                                                         16 * ((2 * ks + h) ^ swz(c))));
    const char* p = O + (8 * h + (ti >> 2) + 16 * ks) * row_bytes + (tlow ^ (blk << 6));
    typedef __attribute__((address_space(3))) s16x4_t* tptr;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)(lds_ptr)p);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)(lds_ptr)(p + 4 * row_bytes));
    const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
    return as_bf16x8(u32x4_t{l2.x, l2.y, h2.x, h2.y});
  };
  auto products = [&](const char* S, const char* SC, int sub) {
    if constexpr (NMB > 0) {
      if constexpr (!F8) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          bf16x8_t mf[NA], jf[NB];
#pragma unroll
          for (int j = 0; j < NB; ++j) jf[j] = frag(S + kM, j0 + j, ks, JT, 2 * TJ);
#pragma unroll
          for (int i = 0; i < NA; ++i) mf[i] = frag(S, m0 + i, ks, MT, 2 * TM);
#pragma unroll
          for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = mfma32x32x16(jf[j], mf[i], acc[i][j]);
        }
      } else {
        uint32_t ms[NA], js[NB];
#pragma unroll
        for (int i = 0; i < NA; ++i)
          ms[i] = *reinterpret_cast<const uint32_t*>(SC + 16 * (32 * (m0 + i) + c) + 4 * sub) >>
                  (8 * h);
#pragma unroll
        for (int j = 0; j < NB; ++j)
          js[j] = *reinterpret_cast<const uint32_t*>(SC + 16 * (TM + 32 * (j0 + j) + c) +
                                                     4 * sub) >>
                  (8 * h);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          i32x8_t mf[NA], jf[NB];
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            const int r = 32 * (j0 + j) + c;
            const i32x4_t v = *reinterpret_cast<const i32x4_t*>(
                S + kM + 64 * r + 16 * ((2 * s + h) ^ ((r >> 2) & 3)));
            jf[j] = i32x8_t{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
          }
#pragma unroll
          for (int i = 0; i < NA; ++i) {
            const char* p = S + 4096 * (m0 + i) + 128 * c;
            const i32x4_t lo =
                *reinterpret_cast<const i32x4_t*>(p + 16 * ((4 * s + h) ^ swz(c)));
            const i32x4_t hi =
                *reinterpret_cast<const i32x4_t*>(p + 16 * ((4 * s + 2 + h) ^ swz(c)));
            mf[i] = i32x8_t{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          }
#pragma unroll
          for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
              if (s == 0)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                    jf[j], mf[i], acc[i][j], 4, 0, 0, js[j], 0, ms[i]);
              else
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                    jf[j], mf[i], acc[i][j], 4, 0, 2, js[j], 2, ms[i]);
            }
        }
      }
    }
  };

  find_x(0);
  if (T > 0) {
    issue(0, smem);
    if (F8) issue_scales(0, scl);
    find_x(1);
  }
  for (int t = 0; t < T; ++t) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < T) {
      issue(t + 1, smem + ((t + 1) & 1) * kStage<KIND, TM, TJ>);
      if (F8 && ((t + 1) & 3) == 0)
        issue_scales((t + 1) >> 2, scl + (((t + 1) >> 2) & 1) * kScales<KIND, TM, TJ>);
      find_x(t + 2);
    }
    products(smem + (t & 1) * kStage<KIND, TM, TJ>,
             scl + ((t >> 2) & 1) * kScales<KIND, TM, TJ>, t & 3);
  }
  __syncthreads();

  // ---- out, 32 rows at a time through the wave's own LDS: lane (c, h) holds output row
  // c and columns 8 q + 4 h .. + 3 of each 32; rows leave by 16-byte stores
  if constexpr (NMB > 0) {
    constexpr int WC = 32 * NB;  // the wave's columns
    char* O = smem + wave * (32 * (4 * WC + 16));
    const int wcol0 = col0 + 32 * j0;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row1 = 32 * (m0 + i);
      const int es = a.out_f32 ? 4 : 2, stride = WC * es + 16;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4_t v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                          acc[i][j][4 * q + 3]};
          char* p = O + c * stride + (32 * j + 8 * q + 4 * h) * es;
          if (a.out_f32)
            *reinterpret_cast<f32x4_t*>(p) = v;
          else
            *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        }
      wave_sync();
      const int cpr = WC * es / 16;  // 16-byte runs a row
      const int64_t obase =
          (KIND == kDw ? (int64_t)e * a.C + row0 : slot0 + row0) * (int64_t)a.J;
      for (int id = lane; id < 32 * cpr; id += 64) {
        const int r = id / cpr, cc = id - r * cpr;
        const int col = wcol0 + cc * 16 / es;
        if (row1 + r < rows && col < a.J)
          *(gptr<u32x4_t>)(as_global<char>(a.out) +
                           (obase + (int64_t)(row1 + r) * a.J + col) * es) =
              *reinterpret_cast<const u32x4_t*>(O + r * stride + 16 * cc);
      }
      wave_sync();
    }
  }
}

// Rows that no group has: zeros.
__device__ __forceinline__ void zero_rows(const GroupedArgs& a, int64_t slot0, int rows, int col0,
                                          int cols) {
  const int es = a.out_f32 ? 4 : 2;
  const int n = min(cols, a.J - col0) * es / 16;  // 16-byte runs a row
  for (int id = threadIdx.x; id < rows * n; id += blockDim.x) {
    const int r = id / n, cc = id - r * n;
    *(gptr<u32x4_t>)(as_global<char>(a.out) + ((slot0 + r) * (int64_t)a.J + col0) * es + 16 * cc) =
        u32x4_t{0, 0, 0, 0};
  }
}

template <int KIND, int TM, int TJ, int WM, int WJ, int STAGES>
__global__ __launch_bounds__(64 * WM * WJ, 2) void grouped_tile_kernel(GroupedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int MB = TM / WM / 32;
  int e, row0 = 0, rows, tj;
  int64_t slot0, len = 0;
  if constexpr (KIND == kDw) {
    const int units = a.E * a.tiles_m * a.tiles_j;
    const int per_x = (units + (int)kXcds - 1) / (int)kXcds;
    const int b = blockIdx.x, u = (b % (int)kXcds) * per_x + b / (int)kXcds;
    if (b / (int)kXcds >= per_x || u >= units) return;
    const int tile = u / a.tiles_j;
    tj = u - tile * a.tiles_j;
    e = tile / a.tiles_m;
    row0 = (tile - e * a.tiles_m) * TM;
    rows = min(TM, a.C - row0);
    slot0 = group_at(a, e);
    len = max(group_at(a, e + 1) - slot0, (int64_t)0);
  } else {
    GroupedTile t;
    if (!find_tile<TM>(a, blockIdx.x, t, tj)) return;
    if (t.e == a.E) {
      zero_rows(a, t.slot0, (int)t.rows, tj * TJ, TJ);
      return;
    }
    e = t.e, slot0 = t.slot0, rows = (int)t.rows;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // 32-row blocks that hold rows of this wave's
  const int nmb = min(max((rows + 31) / 32 - (wave / WJ) * MB, 0), MB);
#define MLXR_GT_UNIT(N) \
  tile_unit<KIND, TM, TJ, WM, WJ, STAGES, N>(a, e, slot0, len, row0, rows, tj * TJ, smem)
  if constexpr (MB == 4) {
    if (nmb == 4)
      MLXR_GT_UNIT(4);
    else if (nmb == 3)
      MLXR_GT_UNIT(3);
    else if (nmb == 2)
      MLXR_GT_UNIT(2);
    else if (nmb == 1)
      MLXR_GT_UNIT(1);
    else
      MLXR_GT_UNIT(0);
  } else {
    static_assert(MB == 2, "wave tiles of 64 or 128 rows");
    if (nmb == 2)
      MLXR_GT_UNIT(2);
    else if (nmb == 1)
      MLXR_GT_UNIT(1);
    else
      MLXR_GT_UNIT(0);
  }
#undef MLXR_GT_UNIT
}

template <int KIND, int TM, int TJ, int WM, int WJ, int STAGES>
hipError_t run_tiles(GroupedArgs a, hipStream_t s) {
  constexpr int lds = kTileLds<KIND, TM, TJ, STAGES>;
  static_assert(lds <= 160 * 1024 && WM * WJ * 32 * (4 * (TJ / WJ) + 16) <= lds, "LDS");
  a.tiles_j = (a.J + TJ - 1) / TJ;
  a.tiles_m = KIND == kDw ? (a.C + TM - 1) / TM : 0;
  const int64_t units = KIND == kDw ? (int64_t)a.E * a.tiles_m * a.tiles_j
                                    : grouped_tiles(a.R, a.E, TM) * a.tiles_j;
  if (units <= 0) return hipSuccess;
  const int64_t grid = (units + kXcds - 1) / kXcds * kXcds;
  if (grid * 64 * WM * WJ > UINT32_MAX) return hipErrorInvalidValue;  // (the callers check)
  grouped_tile_kernel<KIND, TM, TJ, WM, WJ, STAGES>
      <<<(unsigned)grid, 64 * WM * WJ, lds, s>>>(a);
  return hipGetLastError();
}

// Rows a group, from which 256-row tiles are taken instead of 64-row ones.
bool tall(int64_t R, int64_t E) { return R >= 96 * E; }

}  // namespace

hipError_t launch_grouped_mm(const GroupedArgs& a, hipStream_t s) {
  ProfileScope prof("grouped_mm", s);
  return tall(a.R, a.E) ? run_tiles<kForward, 256, 256, 2, 4, 2>(a, s)
                        : run_tiles<kForward, 64, 256, 1, 4, 2>(a, s);
}
hipError_t launch_grouped_dx(const GroupedArgs& a, hipStream_t s) {
  ProfileScope prof("grouped_dx", s);
  return tall(a.R, a.E) ? run_tiles<kDx, 256, 256, 2, 4, 2>(a, s)
                        : run_tiles<kDx, 64, 256, 1, 4, 2>(a, s);
}
hipError_t launch_grouped_dw(const GroupedArgs& a, hipStream_t s) {
  ProfileScope prof("grouped_dw", s);
  return tall(a.R, a.E) ? run_tiles<kDw, 256, 256, 2, 4, 2>(a, s)
                        : run_tiles<kDw, 128, 128, 2, 2, 2>(a, s);
}
hipError_t launch_grouped_qmm(const GroupedArgs& a, hipStream_t s) {
  ProfileScope prof("grouped_qmm", s);
  return tall(a.R, a.E) ? run_tiles<kForward8, 256, 256, 2, 4, 2>(a, s)
                        : run_tiles<kForward8, 64, 256, 1, 4, 2>(a, s);
}

}  // namespace mlxr_moe
