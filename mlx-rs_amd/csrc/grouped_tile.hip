// Products grouped by expert over ragged groups of rows, in tiles on the matrix cores:
//   forward   y[r, n]     = sum_k x[r, k] W[e(r)][n, k]
//   dx        dx[r, k]    = sum_n dy[r, n] W[e(r)][n, k]
//   dW        dW[e][n, k] = sum_{r of e} dy[r, n] x[r, k]
// in bf16 with f32 sums, and the forward product of e4m3 rows by e2m1 weights, each
// with a power-of-two scale per 32 (modes mxfp8 and mxfp4).
//
// One kernel body.  An output tile is TM x TJ; a stage of SI inputs of both operands goes
// straight to LDS by 16-byte loads while the stages before are multiplied.  An operand whose
// inputs run along memory (x and W forward, dy of dx) lies in LDS as rows of a stage's inputs;
// one whose inputs run across rows (W of dx, both of dW) as rows of columns, read transposed by
// ds_read_b64_tr_b16.
//
// Measured (one MI355X; c2: 128 experts, 4096 tokens of 8 choices, 768 x 2048): down 181 us,
// its bytes at a copy's rate 122; dx 202 and 122, dW 253-261 and 98; 8 by 4 bits up 86, floor
// 36; 256 experts of 512 x 2048, 2048 tokens of 8 choices 134, floor 117.  With 4 to 32 equal
// groups 770-910 TFLOP/s.  What bounds the ragged ones: loads and their barriers (of c2 down's
// 198 us by the profiler's clock 195 are left without matrix instructions, 110 without loads),
// and the workgroups' starts and ends (40 with no stage in between).
#include <algorithm>
#include <type_traits>

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

// A stage has SI inputs: bytes of a row of either operand that runs along them ...
template <int KIND, int SI>
constexpr int kMRow = KIND == kForward8 ? SI : 2 * SI;
template <int KIND, int SI>
constexpr int kJRow = KIND == kForward8 ? SI / 2 : 2 * SI;
// ... and of both operands (as much where they run across rows)
template <int KIND, int TM, int TJ, int SI>
constexpr int kStage = TM * kMRow<KIND, SI> + TJ * kJRow<KIND, SI>;
// 8-bit: the scales of 512 inputs, 16 bytes a row, twice.  dW: indices of x's rows.
constexpr int kIndexRows = 512;
template <int KIND, int TM, int TJ>
constexpr int kExtra = KIND == kForward8 ? 2 * 16 * (TM + TJ) : KIND == kDw ? 2 * 4 * kIndexRows
                                                                            : 0;
template <int KIND, int TM, int TJ, int SI, int STAGES>
constexpr int kTileLds = STAGES * kStage<KIND, TM, TJ, SI> + kExtra<KIND, TM, TJ>;

// Waves a SIMD: of as many workgroups as LDS holds (two at most)
template <int KIND, int TM, int TJ, int WM, int WJ, int SI, int STAGES>
constexpr int kWavesPerSimd = std::max(
    1, WM * WJ / 4 * (2 * kTileLds<KIND, TM, TJ, SI, STAGES> <= 160 * 1024 ? 2 : 1));
// LDS that a wave's output rows pass through, 32 at a time
template <int TJ, int WJ>
constexpr int kOutBytes = 32 * (4 * (TJ / WJ) + 16);

// An operand in rows of P 16-byte pieces: piece p of row r lies at p ^ rkey<P>(r), so that
// the 16 rows that a quarter of a wave reads a piece of lie in all 256 bytes of the banks.
template <int P>
__device__ __forceinline__ int rkey(int r) {
  return (r / (16 / P)) & (P - 1);
}
// A transposed operand: 32-byte piece p of row r at p ^ tkey(r).  The four rows and the two
// neighbouring pieces that half a wave reads at once lie in eight different eighths of 256
// bytes so.
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
// The workgroup's barrier, when at most N of this wave's loads are not back and its reads
// and writes of LDS are.
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A tile's place.
struct TileAt {
  int e;           // expert
  int64_t slot0;   // forward, dx: the tile's first sorted row.  dW: the first summed over
  int64_t len;     // dW: sorted rows summed over
  int row0, rows;  // dW: output rows.  Else 0 and the tile's sorted rows
  int col0;        // first column
  void* out;       // of column 0 of the tile's first row
  bool f32;
};

template <int KIND, int TM, int TJ, int WM, int WJ, int SI, int STAGES, int NMB>
__device__ __forceinline__ void tile_unit(const GroupedArgs& a, const TileAt& at, char* smem) {
  constexpr bool F8 = KIND == kForward8, MT = kMTrans<KIND>, JT = kJTrans<KIND>;
  constexpr int NW = WM * WJ;
  constexpr int MB = TM / WM / 32, NB = TJ / WJ / 32;  // 32 x 32 blocks of a wave
  constexpr int NA = NMB > 0 ? NMB : 1;
  constexpr int MR = kMRow<KIND, SI>, JR = kJRow<KIND, SI>;
  constexpr int MP = MT ? TM / 8 : MR / 16, JP = JT ? TJ / 8 : JR / 16;  // pieces a row
  constexpr int kM = TM * MR, kS = kStage<KIND, TM, TJ, SI>;
  constexpr int ML = kM / 1024 / NW, JL = TJ * JR / 1024 / NW;  // loads a wave and stage
  static_assert(ML >= 1 && JL >= 1 && MB >= 1 && NB >= 1 && SI % 32 == 0, "tile");
  static_assert((!MT || TM >= 128) && (!JT || TJ >= 128), "eight 32-byte pieces a row");
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WJ, wj = wave % WJ;
  const int c = lane & 31, h = lane >> 5;
  const int rows = at.rows;

  // ---- where the operands start, how far apart their rows are, how many stages
  const int64_t ldm = F8 ? (int64_t)a.C : (int64_t)a.C * 2;  // bytes
  const int64_t ldj = JT ? (int64_t)a.J * 2 : F8 ? (int64_t)a.C / 2 : (int64_t)a.C * 2;
  const bool mapped = a.rows != nullptr;  // x's rows (M forward, J of dW)
  // (negative indices are past all rows as unsigned ones)
  const uint32_t x_rows = (uint32_t)min(a.x_rows, (int64_t)1 << 31);
  const int T = (int)(((MT ? at.len : a.C) + SI - 1) / SI);
  char* extra = smem + STAGES * kS;

  // ---- the rows' indices: asked for first, waited for behind the first loads of J (a wait
  // for the last load asked for is one for all before it)
  const auto mrow = [&](int i) { return (wave * ML + i) * (64 / MP) + lane / MP; };
  constexpr bool kMap = KIND == kForward || F8;
  int xi[ML] = {}, sx = 0, oi[NA] = {};  // (oi: of the output rows that the lane has)
  const int srow = 64 * wave + lane;  // 8-bit: the row (of x, then of W) whose scales it loads
  if (kMap && mapped) {
#pragma unroll
    for (int i = 0; i < ML; ++i)
      xi[i] = as_global<const int32_t>(a.rows)[at.slot0 + min(mrow(i), rows - 1)];
    if (F8) sx = as_global<const int32_t>(a.rows)[at.slot0 + min(srow, rows - 1)];
#pragma unroll
    for (int i = 0; i < NMB; ++i)
      oi[i] = as_global<const int32_t>(a.rows)[at.slot0 + min(32 * (wm + WM * i) + c, rows - 1)];
  }
  uint64_t none[NA] = {};  // by lane: whether its index names no row of x

  // ---- M
  const char* mp = static_cast<const char*>(a.m);
  int64_t mbytes;
  uint32_t moff[ML];
  if constexpr (MT) {
    mp += at.slot0 * ldm + 2 * (int64_t)at.row0;
    mbytes = at.len * ldm - 2 * (int64_t)at.row0;
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      const int r = mrow(i), p = lane % MP;
      moff[i] = (uint32_t)(r * ldm) + 32 * ((p >> 1) ^ tkey(r)) + 16 * (p & 1);
    }
  } else {
    const bool map = mapped && kMap;
    if (!map) mp += at.slot0 * ldm;
    mbytes = map ? a.x_rows * ldm : rows * ldm;
  }
  const auto place_m = [&] {
    if constexpr (!MT) {
#pragma unroll
      for (int i = 0; i < ML; ++i) {
        const int r = mrow(i), x = kMap && mapped ? xi[i] : r;
        const bool ok = r < rows && (!(kMap && mapped) || (uint32_t)x < x_rows);
        moff[i] = ok ? (uint32_t)x * (uint32_t)ldm + 16 * ((lane % MP) ^ rkey<MP>(r)) : kPastEnd;
      }
    }
    if constexpr (kMap) {
      if (mapped)
#pragma unroll
        for (int i = 0; i < NMB; ++i) none[i] = __ballot((uint32_t)oi[i] >= x_rows);
    }
  };
  // ---- J
  const char* jp = static_cast<const char*>(a.j);
  int64_t jbytes;
  uint32_t joff[JL];
  const auto jrow = [&](int i) { return (wave * JL + i) * (64 / JP) + lane / JP; };
  if constexpr (JT) {
    const bool map = KIND == kDw && mapped;
    jp += 2 * (int64_t)at.col0 +
          (KIND == kDw ? (map ? 0 : at.slot0 * ldj) : (int64_t)at.e * a.C * ldj);
    jbytes = (KIND == kDw ? (map ? a.x_rows : at.len) : (int64_t)a.C) * ldj - 2 * (int64_t)at.col0;
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      const int r = jrow(i), p = lane % JP;
      joff[i] = (map ? 0u : (uint32_t)(r * ldj)) + 32 * ((p >> 1) ^ tkey(r)) + 16 * (p & 1);
    }
  } else {
    jp += ((int64_t)at.e * a.J + at.col0) * ldj;
    jbytes = (int64_t)(a.J - at.col0) * ldj;
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      const int r = jrow(i);
      joff[i] = (uint32_t)(r * ldj) + 16 * ((lane % JP) ^ rkey<JP>(r));
    }
  }
  // ---- dW: kIndexRows indices of x's rows from sorted row q kIndexRows of the group on,
  // straight to LDS (past the rows 0, of rows that are not read)
  auto issue_index = [&](int q) {
    if constexpr (KIND == kDw) {
      const int64_t from = (int64_t)q * kIndexRows;
      const __amdgpu_buffer_rsrc_t r =
          rsrc(reinterpret_cast<const char*>(a.rows + at.slot0 + from), 4 * (at.len - from));
      for (int i = wave; i < kIndexRows / 64; i += NW)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (lds_ptr)(extra + 4 * kIndexRows * (q & 1) + 256 * i), 4, 256 * i + 4 * lane, 0, 0,
            0);
    }
  };
  // ... of stage t's rows (past the last stage of any: nothing of it is read)
  const auto stage_index = [&](int t) {
    return reinterpret_cast<const int*>(extra) + t * SI % (2 * kIndexRows);
  };
  // ---- 8-bit: the scales of inputs 512 q .. 512 q + 511, 16 bytes a row
  const int G = a.C / 32;
  auto issue_scales = [&](int q) {
    if constexpr (F8) {
      char* S = extra + 16 * (TM + TJ) * (q & 1);
      if ((G & 3) == 0) {
        // by aligned words, 64 rows a load
        const __amdgpu_buffer_rsrc_t mr =
            rsrc(reinterpret_cast<const char*>(a.ms) + (mapped ? 0 : at.slot0 * G) + 16 * q,
                 (mapped ? a.x_rows : rows) * (int64_t)G - 16 * q);
        const __amdgpu_buffer_rsrc_t jr =
            rsrc(reinterpret_cast<const char*>(a.js) + ((int64_t)at.e * a.J + at.col0) * G + 16 * q,
                 (int64_t)(a.J - at.col0) * G - 16 * q);
        static_assert(!F8 || (TM + TJ) / 64 <= NW, "one load a wave");
        if (wave < (TM + TJ) / 64) {
          const bool isj = wave >= TM / 64;
          uint32_t off = (uint32_t)(srow - (isj ? TM : 0)) * G;
          if (!isj && mapped) off = (uint32_t)sx < x_rows ? (uint32_t)sx * G : kPastEnd;
          if (!isj && srow >= rows) off = kPastEnd;
          load_lds(isj ? jr : mr, S + 1024 * wave, off);
        }
      } else {
        // rows at any address, byte by byte; zeros past the row
        for (int r = tid; r < TM + TJ; r += 64 * NW) {
          const uint8_t* p = nullptr;
          if (r >= TM) {
            if (at.col0 + r - TM < a.J) p = a.js + ((int64_t)at.e * a.J + at.col0 + r - TM) * G;
          } else if (r < rows) {
            int64_t x = at.slot0 + r;
            if (mapped) x = as_global<const int32_t>(a.rows)[x];
            if (x >= 0 && x < a.x_rows) p = a.ms + x * G;
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
    }
  };

  // ---- a stage's loads, always as many (past the last stage of nothing)
  const int mpieces = (int)(ldm / 16), jpieces = (int)(ldj / 16);
  bool named[ML];
  for (int i = 0; i < ML; ++i) named[i] = true;
  auto issue_m = [&](int t, char* S) {
    if (F8 && t % (512 / SI) == 0 && t < T) issue_scales(t / (512 / SI));
    const int64_t mo = MT ? (int64_t)t * SI * ldm : (int64_t)t * MR;
    const __amdgpu_buffer_rsrc_t mr = rsrc(mp + mo, t < T ? mbytes - mo : 0);
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      bool ok = KIND != kDw || named[i];
      if constexpr (!MT) ok = MP * t + ((lane % MP) ^ rkey<MP>(mrow(i))) < mpieces;
      load_lds(mr, S + (wave * ML + i) * 1024, ok ? moff[i] : kPastEnd);
    }
  };
  // dW: which of this lane's rows of stage t name a row of x.  dy of one that does not is left
  // out as its x is (it may hold a NaN).  Asked for a step ahead: c2's up projection 253 us so,
  // 257 with the look at the loads (247 without any).
  auto look_m = [&](int t) {
    if constexpr (KIND == kDw) {
      if (!mapped) return;
      const int* xi = stage_index(t);
#pragma unroll
      for (int i = 0; i < ML; ++i) {
        named[i] = (uint32_t)xi[mrow(i)] < x_rows;
      }
    }
  };
  auto issue_j = [&](int t, char* S) {
    if constexpr (KIND == kDw) {
      if (mapped) {
        constexpr int kPer = kIndexRows / SI;  // stages a part of the indices
        if (t % kPer == 0 && t > 0) issue_index(t / kPer + 1);
        const __amdgpu_buffer_rsrc_t jr = rsrc(jp, t < T ? jbytes : 0);
        const int* xi = stage_index(t);
#pragma unroll
        for (int i = 0; i < JL; ++i) {
          const uint32_t x = xi[jrow(i)];
          const bool ok = x < x_rows && t * SI + jrow(i) < (int)at.len;
          load_lds(jr, S + kM + (wave * JL + i) * 1024,
                   ok ? joff[i] + x * (uint32_t)ldj : kPastEnd);
        }
        return;
      }
    }
    const int64_t jo = JT ? (int64_t)t * SI * ldj : (int64_t)t * JR;
    const __amdgpu_buffer_rsrc_t jr = rsrc(jp + jo, t < T ? jbytes - jo : 0);
#pragma unroll
    for (int i = 0; i < JL; ++i) {
      bool ok = true;
      if constexpr (!JT) ok = JP * t + ((lane % JP) ^ rkey<JP>(jrow(i))) < jpieces;
      load_lds(jr, S + kM + (wave * JL + i) * 1024, ok ? joff[i] : kPastEnd);
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
  // the wave's blocks: rows 32 (wm + WM i), so that a short tile's are spread over the
  // waves; columns 32 (j0 + j)
  const int j0 = wj * NB;
  // transposed: byte of the lane's four values of block 0, rows 8 h + (lane % 16) / 4
  const int ti = lane & 15, tg = (lane >> 4) & 1;
  const int tlow = ((tg ^ tkey(ti >> 2)) << 5) + 8 * (ti & 3);
  const auto trans = [&](const char* O, int blk, int ks, int row_bytes) -> bf16x8_t {
    const char* p = O + (8 * h + (ti >> 2) + 16 * ks) * row_bytes + (tlow ^ (blk << 6));
    typedef __attribute__((address_space(3))) s16x4_t* tptr;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)(lds_ptr)p);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)(lds_ptr)(p + 4 * row_bytes));
    const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
    return as_bf16x8(u32x4_t{l2.x, l2.y, h2.x, h2.y});
  };
  // The operands of a step: 16 inputs, or 64 of the 8- and 4-bit ones and their scales.
  constexpr int KS = SI / (F8 ? 64 : 16);
  static_assert(KS % 2 == 0, "two sets of operands");
  typedef std::conditional_t<F8, i32x8_t, bf16x8_t> Op;
  Op mf[2][NA], jf[2][NB];
  uint32_t ms[2][NA], js[2][NB];
  // of step ks of the stage t at S into set p
  auto read = [&](const char* S, int t, int ks, int p) {
    if constexpr (NMB > 0 && !F8) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if constexpr (JT)
          jf[p][j] = trans(S + kM, j0 + j, ks, 2 * TJ);
        else
          jf[p][j] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(
              S + kM + (32 * (j0 + j) + c) * JR + 16 * ((2 * ks + h) ^ rkey<JP>(c))));
      }
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        if constexpr (MT)
          mf[p][i] = trans(S, wm + WM * i, ks, 2 * TM);
        else
          mf[p][i] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(
              S + (32 * (wm + WM * i) + c) * MR + 16 * ((2 * ks + h) ^ rkey<MP>(c))));
      }
    } else if constexpr (NMB > 0) {
      // lane half h: 4-bit inputs 32 h .. 32 h + 31 of 64; 8-bit ones 16 h .. + 15 and
      // 32 + 16 h .. + 15; the scales of inputs 32 h .. + 31
      if (ks == 0) {
        const char* SC =
            extra + 16 * (TM + TJ) * (t / (512 / SI) & 1) + t % (512 / SI) * (SI / 32);
#pragma unroll
        for (int i = 0; i < NA; ++i)
          ms[0][i] = *reinterpret_cast<const uint32_t*>(SC + 16 * (32 * (wm + WM * i) + c));
#pragma unroll
        for (int j = 0; j < NB; ++j)
          js[0][j] = *reinterpret_cast<const uint32_t*>(SC + 16 * (TM + 32 * (j0 + j) + c));
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const i32x4_t v = *reinterpret_cast<const i32x4_t*>(
            S + kM + (32 * (j0 + j) + c) * JR + 16 * ((2 * ks + h) ^ rkey<JP>(c)));
        jf[p][j] = i32x8_t{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const char* q = S + (32 * (wm + WM * i) + c) * MR;
        const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(q + 16 * ((4 * ks + h) ^ rkey<MP>(c)));
        const i32x4_t hi =
            *reinterpret_cast<const i32x4_t*>(q + 16 * ((4 * ks + 2 + h) ^ rkey<MP>(c)));
        mf[p][i] = i32x8_t{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      }
    }
  };
  // step ks of a stage, from set p
  auto multiply = [&](int ks, int p) {
    if constexpr (NMB > 0) {
      if (F8 && ks == 0) {
        // this half's scales of the stage, at bytes 0 and 2
#pragma unroll
        for (int i = 0; i < NA; ++i) ms[1][i] = ms[0][i] >> (8 * h);
#pragma unroll
        for (int j = 0; j < NB; ++j) js[1][j] = js[0][j] >> (8 * h);
      }
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if constexpr (!F8)
            acc[i][j] = mfma32x32x16(jf[p][j], mf[p][i], acc[i][j]);
          else if (ks == 0)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                jf[p][j], mf[p][i], acc[i][j], 4, 0, 0, js[1][j], 0, ms[1][i]);
          else
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                jf[p][j], mf[p][i], acc[i][j], 4, 0, 2, js[1][j], 2, ms[1][i]);
        }
    }
  };

  if (KIND == kDw && mapped) {
    issue_index(0);
    issue_index(1);
    stage_barrier<0>();
  }
  // ---- The operands of a step are read during the step before it, so a stage's barrier
  // stands before its last step, when all waves have read the stage for good; the stage
  // STAGES ahead then takes its place.  A stage's loads are back when no more are out than
  // the later stages' (what else is loaded on the way only makes it wait for more).
  issue_j(0, smem);
  __builtin_amdgcn_sched_barrier(0);
  place_m();
  look_m(0);
  issue_m(0, smem);
#pragma unroll
  for (int t = 1; t < STAGES; ++t) {
    look_m(t);
    issue_m(t, smem + t * kS);
    issue_j(t, smem + t * kS);
  }
  stage_barrier<(STAGES - 1) * (ML + JL)>();
  read(smem, 0, 0, 0);
  int from = 0, last = (STAGES - 1) * kS;  // this stage's place, the one's before
#pragma nounroll
  for (int t = 0; t < T; ++t) {
    const int next = from + kS < STAGES * kS ? from + kS : 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks == KS - 1) {
        stage_barrier<(STAGES - 2) * (ML + JL)>();
        read(smem + next, t + 1, 0, 0);
        issue_m(t + STAGES, smem + from);
      } else {
        read(smem + from, t, ks + 1, (ks + 1) & 1);
        if (ks == 0) {
          if (t > 0) issue_j(t - 1 + STAGES, smem + last);
          look_m(t + STAGES);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply(ks, ks & 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    last = from;
    from = next;
  }
  // nothing may be on its way to LDS when it is used again
  stage_barrier<0>();

  // ---- out, 32 rows at a time through the wave's own LDS: lane (c, h) holds output row
  // c and columns 8 q + 4 h .. + 3 of each 32; rows leave by 16-byte stores
  if constexpr (NMB > 0) {
    constexpr int WC = 32 * NB;  // the wave's columns
    char* O = smem + wave * kOutBytes<TJ, WJ>;
    const int wcol0 = 32 * j0, cols = a.J - at.col0;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row1 = 32 * (wm + WM * i);
      const int es = at.f32 ? 4 : 2, stride = WC * es + 16;
      // (zeros where no row of x is, whatever W holds)
      const bool zero = kMap && (none[i] >> lane & 1);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4_t v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                    acc[i][j][4 * q + 3]};
          if (zero) v = f32x4_t{0, 0, 0, 0};
          char* p = O + c * stride + (32 * j + 8 * q + 4 * h) * es;
          if (at.f32)
            *reinterpret_cast<f32x4_t*>(p) = v;
          else
            *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        }
      wave_sync();
      const int cpr = WC * es / 16;  // 16-byte runs a row
      for (int id = lane; id < 32 * cpr; id += 64) {
        const int r = id / cpr, cc = id - r * cpr;
        const int col = wcol0 + cc * 16 / es;
        if (row1 + r < rows && col < cols)
          *(gptr<u32x4_t>)(as_global<char>(at.out) + ((int64_t)(row1 + r) * a.J + col) * es) =
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

__global__ __launch_bounds__(1024) void grouped_plan_kernel(GroupedArgs a) {
  __shared__ int lds[kPlanWords];
  write_plan(a, PlanTeam{}, lds);
}

template <int KIND, int TM, int TJ, int WM, int WJ, int SI, int STAGES>
__global__ __launch_bounds__(64 * WM * WJ, (kWavesPerSimd<KIND, TM, TJ, WM, WJ, SI, STAGES>))
void grouped_tile_kernel(GroupedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int MB = TM / WM / 32;
  constexpr bool DW = KIND == kDw;
  GroupedUnit u;
  if constexpr (DW) {
    const int tiles = a.tiles_m * a.tiles_j, x = blockIdx.x % kXcds, i = blockIdx.x / kXcds;
    const int part = a.plan[x] + i / tiles;
    if (part >= a.plan[x + 1]) return;
    const int4 r = reinterpret_cast<const int4*>(a.plan + kPlanHead)[part];
    u.tile = i % tiles;
    u.e = r.x, u.slot0 = r.y, u.rows = r.z, u.slice = r.w;
  } else {
    int block = blockIdx.x;
    if (KIND == kDx && a.plan) {
      if (block == 0) {
        write_plan(a, PlanTeam{}, reinterpret_cast<int*>(smem));
        return;
      }
      --block;
    }
    // parts go to the XCDs in runs, so that one L2 sees an expert's
    const bool found = find_part<TM>(a, reinterpret_cast<int*>(smem), u, [&](int all, auto& v) {
      const int x = block % (int)kXcds, i = block / (int)kXcds;
      const int part = (int)((int64_t)all * x / kXcds) + i / a.tiles_j;
      v.tile = i % a.tiles_j;
      return part < (int)((int64_t)all * (x + 1) / kXcds) ? part : -1;
    });
    if (!found) return;
    __syncthreads();  // (the stages take the words' place)
  }
  TileAt at;
  at.e = u.e, at.slot0 = u.slot0;
  at.f32 = a.out_f32;
  if constexpr (DW) {
    const int tn = u.tile / a.tiles_j;
    at.len = u.rows;
    at.row0 = tn * TM, at.rows = min(TM, a.C - at.row0);
    at.col0 = (u.tile - tn * a.tiles_j) * TJ;
    // a part of a group of several: its sums in f32, to be joined
    int64_t first = ((int64_t)at.e * a.C + at.row0) * a.J + at.col0;
    at.out = a.out;
    if (u.slice >= 0) {
      if (u.slice >= a.slices) return;
      first = ((int64_t)u.slice * a.C + at.row0) * a.J + at.col0;
      at.out = a.parts;
      at.f32 = true;
    }
    at.out = static_cast<char*>(at.out) + first * (at.f32 ? 4 : 2);
  } else {
    at.len = 0, at.row0 = 0, at.rows = u.rows;
    at.col0 = u.tile * TJ;
    if (u.e == a.E) {
      zero_rows(a, u.slot0, u.rows, at.col0, TJ);
      return;
    }
    at.out = static_cast<char*>(a.out) + ((int64_t)u.slot0 * a.J + at.col0) * (at.f32 ? 4 : 2);
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // 32-row blocks that hold rows of this wave's
  const int nmb = max((at.rows + 31) / 32 - wave / WJ + WM - 1, 0) / WM;
#define MLXR_GT_UNIT(N) tile_unit<KIND, TM, TJ, WM, WJ, SI, STAGES, N>(a, at, smem)
  if constexpr (MB == 2) {
    if (nmb == 2)
      MLXR_GT_UNIT(2);
    else if (nmb == 1)
      MLXR_GT_UNIT(1);
    else
      MLXR_GT_UNIT(0);
  } else {
    static_assert(MB == 1, "wave tiles of 32 or 64 rows");
    if (nmb == 1)
      MLXR_GT_UNIT(1);
    else
      MLXR_GT_UNIT(0);
  }
#undef MLXR_GT_UNIT
}

// The parts of dW of the groups that are summed in several, added in order.  Workgroup b
// takes slice b / kJoinParts' group, if the slice is the group's first, and part b %
// kJoinParts of it.
constexpr int kJoinParts = 64;
__global__ __launch_bounds__(256) void grouped_join_kernel(GroupedArgs a) {
  const int slice = blockIdx.x / kJoinParts;
  const int2 r = reinterpret_cast<const int2*>(a.plan + kPlanHead + 4 * a.max_parts)[slice];
  const int e = r.x, n = r.y;
  if (n <= 1 || slice + n > a.slices) return;
  const int64_t size = (int64_t)a.C * a.J;  // (8 divides it)
  const f32x4_t* p = reinterpret_cast<const f32x4_t*>(a.parts + slice * size);
  const int64_t o = (int64_t)e * size;
  for (int64_t i = (blockIdx.x % kJoinParts) * 256 + threadIdx.x; i < size / 4;
       i += kJoinParts * 256) {
    f32x4_t v = p[i];
    for (int k = 1; k < n; ++k) v += p[k * (size / 4) + i];
    if (a.out_f32)
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + o + 4 * i) = v;
    else
      *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(a.out) + o + 4 * i) =
          u32x2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  }
}

template <int KIND, int TM, int TJ, int WM, int WJ, int SI, int STAGES>
hipError_t run_tiles(GroupedArgs a, hipStream_t s) {
  constexpr int lds = kTileLds<KIND, TM, TJ, SI, STAGES>;
  static_assert(lds <= 160 * 1024 && WM * WJ * kOutBytes<TJ, WJ> <= lds && 4 * kPlanWords <= lds,
                "LDS");
  int64_t grid;
  if constexpr (KIND == kDw) {
    static_assert(TM == kDwTM && TJ == kDwTJ, "the plan's");
    grid = (int64_t)a.max_run * a.tiles_m * a.tiles_j * kXcds;
  } else {
    a.tiles_j = (a.J + TJ - 1) / TJ;
    const int64_t parts = grouped_tiles(a.R, a.E, TM);
    grid = (parts + kXcds - 1) / kXcds * a.tiles_j * kXcds + (KIND == kDx && a.plan ? 1 : 0);
  }
  if (grid * 64 * WM * WJ > UINT32_MAX) return hipErrorInvalidValue;  // (the callers check)
  grouped_tile_kernel<KIND, TM, TJ, WM, WJ, SI, STAGES>
      <<<(unsigned)grid, 64 * WM * WJ, lds, s>>>(a);
  return hipGetLastError();
}

// Whether 128-row tiles are left to fill half of the chip, at two workgroups a CU.
bool few_tiles(int64_t R, int64_t E, int64_t J, int64_t TJ) {
  return grouped_tiles(R, E, 128) * ((J + TJ - 1) / TJ) < 256;
}

}  // namespace

// 128 x 256 tiles by eight waves, two workgroups a CU (128 registers a lane): of the tiles
// that fit the best in all but the smallest calls.  At c2's down projection over 32768 rows
// (128 experts, J 2048, C 768; these and the next before steps that took a few us off each):
// 185 us, 256 x 256 200, 256 x 128 214, 128 x 128 by four waves 203; dx of its up projection
// 206, 224, 242, 234.
//
// 64 x 128 by four waves where these are few: 1024 rows of 8 experts, J 768, C 2048 18.5 us
// against 33.2, its dx 16.6 against 20.6; 4096 rows 25.5 against 35.1, but dx, J 2048, with
// 328 tiles, 43.9 against 26.7.  Forward also where a group has few rows: 64 a group of 256
// experts (J 512, C 2048) 136 us against 147, 96 a group 143 against 129.  (dx reads the
// weights' rows, 256 bytes of them in these tiles: 64 a group 181 us against 130.)
hipError_t launch_grouped_mm(const GroupedArgs& a, hipStream_t s) {
  if (grouped_streams(a)) return launch_grouped_stream(a, s);
  if (a.R <= 64 * (int64_t)a.E || few_tiles(a.R, a.E, a.J, 256))
    return run_tiles<kForward, 64, 128, 1, 4, 64, 3>(a, s);
  return run_tiles<kForward, 128, 256, 2, 4, 32, 3>(a, s);
}
hipError_t launch_grouped_dx(const GroupedArgs& given, const GroupedArgs* dw, hipStream_t s) {
  GroupedArgs a = given;
  if (dw) {
    const GroupedArgs p = with_plan(*dw);
    a.plan = p.plan, a.chunk = p.chunk, a.slices = p.slices;
    a.max_parts = p.max_parts, a.max_run = p.max_run;
  }
  if (few_tiles(a.R, a.E, a.J, 256)) return run_tiles<kDx, 64, 128, 1, 4, 64, 3>(a, s);
  return run_tiles<kDx, 128, 256, 2, 4, 32, 3>(a, s);
}
// (128 x 128 tiles by four waves: 14.9 us against 16.2 at 1527 rows of 13 experts of 424 x
// 1032, 23.1 against 22.9 at 1024 rows of 8 of 768 x 2048, 297 against 269 at c2's.)
hipError_t launch_grouped_dw(const GroupedArgs& given, bool planned, hipStream_t s) {
  const GroupedArgs a = with_plan(given);
  if (!planned) grouped_plan_kernel<<<1, 1024, 0, s>>>(a);
  const hipError_t e = run_tiles<kDw, kDwTM, kDwTJ, 2, 4, 32, 3>(a, s);
  if (e != hipSuccess || !a.slices) return e;
  grouped_join_kernel<<<(unsigned)(a.slices * kJoinParts), 256, 0, s>>>(a);
  return hipGetLastError();
}
// 128 x 128 by four waves, one a SIMD: at c2's up projection over 32768 rows 97 us, 128 x
// 256 by eight 102, 64 x 256 by four 135.  64 x 128 where a group has few rows (16 a group
// of 256 experts, J 512, C 2048: 32.0 us against 35.1; 64: 51 against 46) or the tiles are few
// (1024 rows of 8 experts, J 768: 14.3 against 18.1).
hipError_t launch_grouped_qmm(const GroupedArgs& a, hipStream_t s) {
  if (grouped_streams(a)) return launch_grouped_stream(a, s);
  if (a.R <= 32 * (int64_t)a.E || few_tiles(a.R, a.E, a.J, 128))
    return run_tiles<kForward8, 64, 128, 1, 4, 128, 3>(a, s);
  return run_tiles<kForward8, 128, 128, 2, 2, 128, 3>(a, s);
}

}  // namespace mlxr_moe
