// Grouped expert GEMM of microscaled 4-bit weights for few rows per expert
// (decode).
//
//   out[p, n] = sum_k x[row(p), k] * w[e, n, k]
//
// over work items (at most 8 rows of one expert), f32 sums of exact bf16
// products.  HBM-bound: 4.25 bits a weight, each read once per item.
//
// A workgroup is four waves: one item x (64 / KS) nb channels.  A wave owns nb
// blocks of 16 channels (gated: of gate and of up) over one of KS slices of the
// input dim; the slices' sums meet in LDS, added in slice order.  Per step of four
// groups (128 inputs) lane (n, q) = (l % 16, l / 16) loads the 16 bytes of channel
// n's group 4 s + q and makes four MFMA operands of them: in operand i, quarter q
// holds inputs 8 i .. 8 i + 7 of its group, so x is read from LDS in the same
// order, and one v_mfma_f32_16x16x32_bf16 sums 8 inputs of four groups at once.  A
// lane converts its 32 weights with 16 instructions and one scale.  D steps of
// loads are in flight per wave, across its blocks.  The scale bytes of the wave's
// channels are contiguous in memory and come to LDS whole at the start: a byte
// load per step from each of 16 rows takes the address path as long as the 1 KB of
// weights beside it.
//
// c6 T=7: gate/up 57 MB in 13.8 us, down 28 MB in 9.0; c2 T=16 26.8 + 14.6 us, 5
// TB/s.  (With loads that keep no cache place, half a line is fetched twice: 17 us for
// 14 at c6 T=7.)
//
// The items come from a dispatch's records, or, with up to 64 rows, are found by
// every workgroup for itself from the expert ids (MxIds): ten ballots group a
// wave's ids, which takes less than waiting for a record and saves the dispatch's
// launch.
#include <algorithm>

#include "mx.hpp"
#include "prefill_reg.hpp"
#include "qgemm_stream.hpp"

namespace mlxr_moe {
namespace {

// timing builds: steps in flight (gated, not; four and six: c6 T=7 14.6 us for 13.8 and
// 11.5 for 9.9), and workgroups to keep with two blocks a wave (384: down of c4 T=3 7.7
// us, with 768 9.5)
#ifndef MLXR_MX_DG
#define MLXR_MX_DG 2
#endif
#ifndef MLXR_MX_D
#define MLXR_MX_D 3
#endif
#ifndef MLXR_MX_NB_UNITS
#define MLXR_MX_NB_UNITS 384
#endif
constexpr int kWaves = 4;
typedef __attribute__((address_space(3))) void* lds_ptr;

struct MxShape {
  int tiles_n;  // channel tiles per item
  int nb;       // 16-channel blocks per wave
  int units1, items1, rows2;
  int sc_bytes;  // LDS of a wave's scales, one side (whole KB)
};

// An item: rows [0, nt) of expert e; flat rows in fl, or slots from row0 on.
struct Item {
  int e, nt, row0;
  int fl[kWorkRows];
};

// The item of this workgroup from the ids, each wave for itself: equal ids form
// an expert's rows, every TT-th of them starts an item; items are in the order of
// those.  False without one.  Ids outside [0, E) are no one's: workgroup 0 sets the
// status word (skip_minus1: not for -1), and with zero_bad every first item's
// workgroup clears their rows of its channels [ch0, ch0 + chs).
__device__ __forceinline__ bool find_item(const MxIds& d, int ai, bool status, int ch0, int chs,
                                          uint16_t* out, int64_t out_ld, Item& it) {
  constexpr int TT = kWorkRows;
  const int lane = threadIdx.x & 63;
  const bool row = lane < d.n;
  const int batch = lane / d.M;
  const int id = row ? d.ids[batch] : -1;
  bool ok = row && (uint32_t)id < (uint32_t)d.E;
  if (d.lhs && row) ok = ok && d.lhs[batch] < (uint32_t)d.x_batch;
  uint64_t peers = __ballot(ok);
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    const uint64_t m = __ballot((id >> b) & 1);
    peers &= (id >> b) & 1 ? m : ~m;
  }
  const uint64_t below = (1ull << lane) - 1;
  const int rank = __popcll(peers & below);
  const uint64_t starts = __ballot(ok && rank % TT == 0);
  if (ai == 0) {
    const uint64_t bad = __ballot(row && !ok && !(d.skip_minus1 && id == -1));
    if (status && d.status && threadIdx.x == 0) *d.status = bad != 0;
    const uint64_t all = __ballot(row && !ok);
    if (d.zero_bad && all) {
      for (int r = 0; r < d.n; ++r)
        if ((all >> r) & 1)
          for (int i = threadIdx.x; i < chs; i += 64 * kWaves) out[r * out_ld + ch0 + i] = 0;
    }
  }
  if (ai >= __popcll(starts)) return false;
  // the lane that starts item ai
  const uint64_t mine = __ballot(((starts >> lane) & 1) && __popcll(starts & below) == ai);
  const int s = __ffsll((unsigned long long)mine) - 1;
  const uint32_t rows_hi = (uint32_t)__builtin_amdgcn_readlane((int)(peers >> 32), s);
  const uint32_t rows_lo = (uint32_t)__builtin_amdgcn_readlane((int)peers, s);
  const uint64_t rows = (uint64_t)rows_hi << 32 | rows_lo;
  const int base = __builtin_amdgcn_readlane(rank, s);
  it.e = __builtin_amdgcn_readlane(id, s);
  it.nt = min(__popcll(rows) - base, TT);
  it.row0 = 0;
  const bool in = (rows >> lane) & 1;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const uint64_t m = __ballot(in && rank == base + min(t, it.nt - 1));
    it.fl[t] = __ffsll((unsigned long long)m) - 1;
  }
  return true;
}

template <bool GATED, int KS, int D, bool IDS>
__global__ __launch_bounds__(64 * kWaves, 4) void mx_stream_kernel(
    QGemmArgs a, QGemmArgs a2, MxShape sh, MxIds ids) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NM = GATED ? 2 : 1, TT = kWorkRows;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cw = wave / KS, kq = wave % KS;
  const int n = lane & 15, q = lane >> 4;
  Item it;
  int tile;
  bool second = false;
  if constexpr (IDS) {
    const int ai = blockIdx.x / sh.tiles_n;
    tile = blockIdx.x - ai * sh.tiles_n;
    const int chs = kWaves / KS * sh.nb * 16;
    if (!find_item(ids, ai, blockIdx.x == 0, tile * chs, chs, a.out, a.out_ld, it)) return;
  } else {
    Unit u;
    if (!decode_unit<TT>(a, sh.tiles_n, sh.units1, sh.items1, sh.rows2, u)) return;
    second = u.shared;
    tile = u.tile;
    it.e = u.wk.x, it.row0 = u.wk.y, it.nt = min(u.wk.z, TT);
    const int fl[8] = {u.fr0.x, u.fr0.y, u.fr0.z, u.fr0.w, u.fr1.x, u.fr1.y, u.fr1.z, u.fr1.w};
#pragma unroll
    for (int t = 0; t < TT; ++t) it.fl[t] = t < it.nt ? fl[t] : fl[0];
  }
  const RegArgs r = pick_reg(second, a2, 0, a, 0);
  const int K = a.K, G = K / kMxGroup, S = (G + 3) / 4;
  const int nt = it.nt;
  const int SS = (S + KS - 1) / KS, s0 = kq * SS;
  const int cnt = max(min(S - s0, SS), 0);  // this wave's steps of a block
  const int nb = KS > 1 ? 1 : sh.nb;
  const int total = nb * cnt;
  const int ch0 = (tile * (kWaves / KS) + cw) * nb * 16;  // the wave's channels
  const int64_t wrow0 = (int64_t)it.e * r.e_rows + ch0;
  const u32x4_t* wp[NM];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    const QWeights& W = m == 0 ? r.w0 : r.w1;
    wp[m] = reinterpret_cast<const u32x4_t*>(W.w) + (wrow0 + n) * G;
  }
  const __amdgpu_buffer_rsrc_t sr0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(r.w0.scales) + wrow0 * (G / 2), 0, nb * 16 * G, kBufFlags);
  const __amdgpu_buffer_rsrc_t sr1 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(GATED ? r.w1.scales : r.w0.scales) + wrow0 * (G / 2), 0, nb * 16 * G,
      kBufFlags);
  // LDS: x [TT][xs], the waves' scales, and with slices their sums
  const int xs = 128 * S + 8;  // 16 bytes more a row, so that rows start on other banks
  uint16_t* xl = reinterpret_cast<uint16_t*>(smem);
  const int x_bytes = (TT * xs * 2 + 15) & ~15;
  char* scl = smem + x_bytes + wave * NM * sh.sc_bytes;
#pragma unroll
  for (int m = 0; m < NM; ++m)
    for (int o = 0; o < sh.sc_bytes; o += 1024)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(m ? sr1 : sr0,
                                               (lds_ptr)(scl + m * sh.sc_bytes + o), 16,
                                               o + 16 * lane, 0, 0, 0);
  // x rows: thread k8 holds inputs 8 k8 .. 8 k8 + 7 of every row of the item
  int64_t xr[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    if constexpr (IDS) {
      const int f = it.fl[t], b = f / ids.M;
      xr[t] = (int64_t)(ids.lhs ? (int)ids.lhs[b] : b / ids.div) * ids.M + (f - b * ids.M);
    } else if (r.x_by_slot) {
      xr[t] = it.row0 + min(t, nt - 1);
    } else {
      const int f = it.fl[t];
      xr[t] = r.row_map ? r.row_map[f] : f / r.row_div;
    }
  }
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
        if (t < nt) *reinterpret_cast<u32x4_t*>(xl + t * xs + 8 * k8) = v[t];
    }
  };
  u32x4_t xv[TT];
  load_x(tid, xv);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);

  u32x4_t w[D][NM];
  int pb = 0, ps = 0;  // the next load: block, step within it (the last one again past the end)
  auto load_w = [&](int j) {
    const int64_t at = (int64_t)pb * 16 * G + min(4 * min(s0 + ps, S - 1) + q, G - 1);
#pragma unroll
    for (int m = 0; m < NM; ++m) w[j][m] = wp[m][at];
    if (ps + 1 < cnt)
      ++ps;
    else if (pb + 1 < nb)
      ps = 0, ++pb;
  };
#pragma unroll
  for (int j = 0; j < D; ++j) load_w(j);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  store_x(tid, xv);
  for (int k8 = tid + 64 * kWaves; k8 < per_row; k8 += 64 * kWaves) {
    u32x4_t v[TT];
    load_x(k8, v);
    store_x(k8, v);
  }
  // (the scales were issued before the D * NM weight loads)
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(D * NM) : "memory");
  __syncthreads();

  f32x4_t acc[NM];
#pragma unroll
  for (int m = 0; m < NM; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // (rows past the item's read its first row: their sums go nowhere)
  const uint16_t* xa = xl + (n < nt ? n : 0) * xs + 32 * q;
  const bool ragged = G & 3;  // the last step has groups past the row
  auto finish = [&](int b) {  // block b's sums are whole
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * q + i;
      if (t < nt) {
        const int ch = ch0 + 16 * b + n;
        int64_t orow = it.row0 + t;
        if (IDS || (!GATED && r.out_by_flat)) {
          int f = it.fl[0];
#pragma unroll
          for (int k = 1; k < TT; ++k) f = t == k ? it.fl[k] : f;
          orow = f;
        }
        r.out[orow * r.out_ld + ch] =
            GATED ? mx_bf16(mx_act(r.act, acc[0][i], acc[NM - 1][i])) : mx_bf16(acc[0][i]);
      }
    }
  };
  int cb = 0, cs = 0;  // block and step of the next sum
  for (int g0 = 0; g0 < total; g0 += D) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (g0 + j < total) {
        const int s = s0 + cs;
        bf16x8_t xf[4];
#pragma unroll
        for (int f = 0; f < 4; ++f)
          xf[f] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(xa + 128 * s + 8 * f));
        const int g = min(4 * s + q, G - 1);
        uint32_t b[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m)
          b[m] = *reinterpret_cast<const uint8_t*>(scl + m * sh.sc_bytes + (16 * cb + n) * G + g);
        if (ragged) {  // (x is zero there)
          const bool in = 4 * s + q < G;
#pragma unroll
          for (int m = 0; m < NM; ++m) {
            b[m] = in ? b[m] : 0u;
#pragma unroll
            for (int f = 0; f < 4; ++f) w[j][m][f] = in ? w[j][m][f] : 0u;
          }
        }
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const float scale = mx_scale(b[m]);
#pragma unroll
          for (int f = 0; f < 4; ++f)
            acc[m] = mfma16x16x32(xf[f], mx_weights(w[j][m][f], scale), acc[m]);
        }
        if (++cs == cnt) {
          if constexpr (KS == 1) {
            finish(cb);
#pragma unroll
            for (int m = 0; m < NM; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          }
          cs = 0;
          ++cb;
        }
      }
      load_w(j);
    }
  }

  if constexpr (KS > 1) {
    // the slices' sums, in slice order, on the first slice's wave
    f32x4_t* red = reinterpret_cast<f32x4_t*>(smem + x_bytes + kWaves * NM * sh.sc_bytes);
#pragma unroll
    for (int m = 0; m < NM; ++m) red[(wave * NM + m) * 64 + lane] = acc[m];
    __syncthreads();
    if (kq != 0) return;
#pragma unroll
    for (int k = 1; k < KS; ++k)
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[m] += red[((wave + k) * NM + m) * 64 + lane];
    finish(0);
  }
}

}  // namespace

hipError_t launch_mx_stream(const QGemmArgs& a, int64_t max_items, const QGemmArgs* shared,
                            int64_t shared_rows, const char* profile, hipStream_t s,
                            const MxIds* ids) {
  const QGemmArgs& b = shared ? *shared : a;
  if (a.work_rows != kWorkRows || (!ids && !a.work)) return hipErrorInvalidValue;
  const int64_t items2 = shared ? (shared_rows + kWorkRows - 1) / kWorkRows : 0;
  const int64_t items = max_items + items2;
  const int G = a.K / kMxGroup, S = (G + 3) / 4;
  const int nm = a.gated ? 2 : 1;
  const size_t x_lds = ((size_t)kWorkRows * (128 * S + 8) * 2 + 15) & ~size_t(15);
  // slices of the input dim, four steps each at least, while the workgroups, which
  // all stage the whole x, are no more than four a CU up to K = 2048, two above.  (So many
  // run at once where a product is not gated and x is whole: 37 and 74 KB of LDS.  The
  // limit is a count of workgroups all the same: gated ones take 41 KB at K = 2048 and 82
  // at 4096, so three and one of them fit a CU, and those of a launch near the limit run
  // in rounds.  1, 2 and 4 slices, c5 T=1 up 18, 12.0 and 16.4 us, c5 T=2 up 14.6, 18.3 and
  // 20.8, c2 T=4 gate/up 14.2, 13.7 and 16.8, c2 T=2 10.6 with two and 10.1 with four;
  // shorter slices lose, down of c2 T=1 6.0 and 6.7 with two)
  const int64_t slots = 256 * (x_lds <= 36 * 1024 ? 4 : 2);
  int ks = 1;
  while (ks < kWaves && items * (a.N / 64) * ks * 2 <= slots && S >= 8 * ks) ks *= 2;
  // two blocks a wave where one is short of steps, for the staging of x and the scales
  // to pay, with enough workgroups left: one block then two, down of c4 T=60 (4 steps)
  // 46 us and 38, of c2 T=16 (6) 16.8 and 14.8, of c5 T=2 (12) 13.6 and 12.6, of c5 T=8
  // 34.4 and 34.4; but longer ones make rounds of workgroups long: c4 T=60 gate/up (16)
  // 60 and 63, c5 T=16 up (32) 52 and 67
  const int nb = ks == 1 && S < 16 && a.N % 128 == 0 &&
                         items * (a.N / 128) >= MLXR_MX_NB_UNITS
                     ? 2
                     : 1;
  const int tiles_n = a.N / (16 * (kWaves / ks) * nb);
  const int sc_bytes = (nb * 16 * G + 1023) / 1024 * 1024;
  const size_t lds = x_lds + (size_t)kWaves * nm * sc_bytes +
                     (ks > 1 ? (size_t)kWaves * nm * 64 * sizeof(f32x4_t) : 0);
  const MxShape sh{tiles_n, nb, (int)(max_items * tiles_n), (int)max_items, (int)shared_rows,
                   sc_bytes};
  const dim3 grid((unsigned)(items * tiles_n));
  const MxIds none{};
  ProfileScope prof(profile, s);
#define MLXR_MX(G_, KS_, IDS_)                                                            \
  mx_stream_kernel<G_, KS_, (G_) ? MLXR_MX_DG : MLXR_MX_D, IDS_>                          \
      <<<grid, 64 * kWaves, lds, s>>>(a, b, sh, IDS_ ? *ids : none)
#define MLXR_MX_K(G_, IDS_)   \
  do {                        \
    if (ks == 4)              \
      MLXR_MX(G_, 4, IDS_);   \
    else if (ks == 2)         \
      MLXR_MX(G_, 2, IDS_);   \
    else                      \
      MLXR_MX(G_, 1, IDS_);   \
  } while (0)
#define MLXR_MX_G(IDS_)       \
  do {                        \
    if (a.gated)              \
      MLXR_MX_K(true, IDS_);  \
    else                      \
      MLXR_MX_K(false, IDS_); \
  } while (0)
  if (ids)
    MLXR_MX_G(true);
  else
    MLXR_MX_G(false);
#undef MLXR_MX_G
#undef MLXR_MX_K
#undef MLXR_MX
  return hipGetLastError();
}

}  // namespace mlxr_moe
