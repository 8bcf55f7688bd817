// The router's balance loss, its per-expert counts, and its gradient, on gfx950.
//
// Over T tokens' logits z [T, E] and choices idx [T, K], a token counted while
// its mask is not zero (N of them):
//   p[t, :]  = softmax(z[t, :])
//   counts_e = choices of counted tokens that fell on e
//   probs_e  = sum_t p[t, e] / N
//   loss     = E * sum_e counts_e / (N K) * probs_e
// and, the counts being constants of the loss as usual,
//   dz[t, e] = dloss * E / N * p[t, e] * (f_e - sum_j p[t, j] f_j),  f = counts / (N K)
// plus the gradient of the renormalised top-k weights w[t, :] = softmax of the
// K chosen logits (crates/mlxr-lm/src/qwen3_5/text/moe.rs:136-138),
//   dz[t, idx[t, k]] += w[t, k] * (dw[t, k] - sum_j w[t, j] dw[t, j]).
// A row whose logits are all -inf has no probabilities: it adds none, and its
// gradient is 0 (w alike, over the chosen logits).  NaN or +inf among the logits
// makes their softmax NaN.  With N = 0 everything is 0.
//
// One pass over the logits, a wave per row, in the summation orders fixed here
// (no floating-point atomics): a wave's rows add up in registers, a workgroup's
// waves in LDS, the workgroups' in f64 by a second kernel.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"
#include "nn.hpp"

namespace mlxr_moe {
namespace {

constexpr int kWaves = 4;        // per workgroup of the gradient
constexpr int kPartWaves = 16;   // of the two-launch form's first
constexpr int kSmallWaves = 16;  // of the one-workgroup form
constexpr int kJoinCols = 16;    // experts per workgroup of the second launch
constexpr int kJoinRows = 64;    // partials it reads at a time
constexpr float kLog2e = 1.4426950408889634f;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
// op over the 64 lanes, the same bits on every lane (op commutes)
template <class Op>
__device__ __forceinline__ float wave_all(float v, Op op) {
  v = op(v, dpp<0xB1>(v));   // lane ^ 1
  v = op(v, dpp<0x4E>(v));   // lane ^ 2
  v = op(v, dpp<0x141>(v));  // mirrored in 8: the other four
  v = op(v, dpp<0x140>(v));  // mirrored in 16: the other eight
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float wave_add(float v) {
  return wave_all(v, [](float x, float y) { return x + y; });
}

template <bool BF16>
__device__ __forceinline__ float logit(const void* z, int64_t i) {
  if constexpr (BF16)
    return bf16_to_f32(static_cast<const uint16_t*>(z)[i]);
  else
    return static_cast<const float*>(z)[i];
}

// Row t's logits, lane l holding experts l + 64 j; -inf past E.
template <bool BF16, int SLOTS>
__device__ __forceinline__ void load_row(const void* z, int64_t ld, int64_t t, int E, int lane,
                                         float (&v)[SLOTS]) {
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const int e = lane + 64 * j;
    v[j] = e < E ? logit<BF16>(z, t * ld + e) : -INFINITY;
  }
}
// What the exponents of a softmax are taken against, for logits of maximum m.  fmaxf
// leaves NaN out of a maximum, so one of -inf may hide it behind the -inf of experts
// that are shut off and of lanes past the end: against 0 all of those come to 0 and NaN
// stays NaN, so the sum tells a row of nothing (0) from one of NaN.  (Any other sum is 1
// at least.)
__device__ __forceinline__ float softmax_base(float m) { return m == -INFINITY ? 0.0f : m; }
// v := softmax over the wave (0 everywhere where all logits are -inf).  NaN or +inf
// make the row NaN.
template <int SLOTS>
__device__ __forceinline__ void softmax_row(float (&v)[SLOTS]) {
  float m = v[0];
#pragma unroll
  for (int j = 1; j < SLOTS; ++j) m = fmaxf(m, v[j]);
  m = softmax_base(wave_max(m));
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    v[j] = __builtin_amdgcn_exp2f((v[j] - m) * kLog2e);
    s += v[j];
  }
  s = wave_add(s);
  const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) v[j] *= inv;
}

struct BalanceArgs {
  const void* z;
  int64_t ld, T;
  int E, K;
  const int32_t* idx;
  const uint8_t* mask;  // null: every token counts
};

// One workgroup's rows [r0, r1): the sums of their probabilities in red
// [waves, E], the counts in hist [E], (counted rows, bad indices) in tally [2].
template <bool BF16, int SLOTS, int WAVES>
__device__ __forceinline__ void sum_rows(const BalanceArgs& a, int64_t r0, int64_t r1, float* red,
                                         int* hist, int* tally) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int e = tid; e < a.E; e += 64 * WAVES) hist[e] = 0;
  if (tid < 2) tally[tid] = 0;
  __syncthreads();
  float acc[SLOTS];
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) acc[j] = 0.0f;
  int kept = 0;
  for (int64_t t = r0 + wave; t < r1; t += WAVES) {
    if (a.mask && a.mask[t] == 0) continue;
    ++kept;
    float v[SLOTS];
    load_row<BF16, SLOTS>(a.z, a.ld, t, a.E, lane, v);
    softmax_row<SLOTS>(v);
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) acc[j] += v[j];
  }
  // the choices: integers, any order
  bool bad = false;
  for (int64_t i = r0 * a.K + tid; i < r1 * a.K; i += 64 * WAVES) {
    if (a.mask && a.mask[i / a.K] == 0) continue;
    const uint32_t e = (uint32_t)a.idx[i];
    if (e < (uint32_t)a.E)
      atomicAdd(&hist[e], 1);
    else
      bad = true;
  }
  if (bad) tally[1] = 1;
  if (lane == 0 && kept) atomicAdd(&tally[0], kept);
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const int e = lane + 64 * j;
    if (e < a.E) red[wave * a.E + e] = acc[j];
  }
  __syncthreads();
}

// Per workgroup: partial sums [G, E], counts [G, E], tallies [G, 2]; and the
// second launch's ticket.
template <bool BF16, int SLOTS>
__global__ __launch_bounds__(64 * kPartWaves) void balance_part_kernel(
    BalanceArgs a, int rows, float* __restrict__ sums, int32_t* __restrict__ cnts,
    int32_t* __restrict__ tallies, int32_t* __restrict__ ticket) {
  extern __shared__ float lds[];
  float* red = lds;
  int* hist = reinterpret_cast<int*>(red + kPartWaves * a.E);
  int* tally = hist + a.E;
  const int64_t r0 = (int64_t)blockIdx.x * rows;
  sum_rows<BF16, SLOTS, kPartWaves>(a, r0, min(r0 + rows, a.T), red, hist, tally);
  for (int e = threadIdx.x; e < a.E; e += 64 * kPartWaves) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kPartWaves; ++w) s += red[w * a.E + e];
    sums[(int64_t)blockIdx.x * a.E + e] = s;
    cnts[(int64_t)blockIdx.x * a.E + e] = hist[e];
  }
  if (threadIdx.x < 2) tallies[2 * blockIdx.x + threadIdx.x] = tally[threadIdx.x];
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
}

// kJoinCols experts a workgroup: their partials summed in f64, kJoinRows of the
// workgroups at a time.  The workgroup that finishes last adds up the others'
// shares of the loss, in their order.
__global__ __launch_bounds__(kJoinCols* kJoinRows) void balance_join_kernel(
    int G, int E, int K, const float* __restrict__ sums, const int32_t* __restrict__ cnts,
    const int32_t* __restrict__ tallies, double* __restrict__ shares,
    int32_t* __restrict__ ticket, float* __restrict__ loss, int32_t* __restrict__ counts,
    float* __restrict__ probs, int32_t* __restrict__ tokens, int32_t* __restrict__ status) {
  __shared__ double s_l[kJoinRows][kJoinCols];
  __shared__ int c_l[kJoinRows][kJoinCols], n_l[2], last;
  const int tid = threadIdx.x, col = tid % kJoinCols, row = tid / kJoinCols;
  const int e = blockIdx.x * kJoinCols + col;
  if (tid < 2) n_l[tid] = 0;
  __syncthreads();
  double s = 0.0;
  int c = 0;
  if (e < E) {
    constexpr int U = 4;  // partials in flight
    for (int g0 = row; g0 < G; g0 += U * kJoinRows) {
      float sv[U];
      int cv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = (int64_t)min(g0 + u * kJoinRows, G - 1) * E + e;
        sv[u] = sums[at], cv[u] = cnts[at];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (g0 + u * kJoinRows < G) s += sv[u], c += cv[u];
    }
  }
  int n = 0, bad = 0;
  for (int g = tid; g < G; g += kJoinCols * kJoinRows)
    n += tallies[2 * g], bad |= tallies[2 * g + 1];
  if (n) atomicAdd(&n_l[0], n);
  if (bad) n_l[1] = 1;
  s_l[row][col] = s;
  c_l[row][col] = c;
  __syncthreads();
#pragma unroll
  for (int m = kJoinRows / 2; m > 0; m >>= 1) {
    if (row < m) {
      s_l[row][col] += s_l[row + m][col];
      c_l[row][col] += c_l[row + m][col];
    }
    __syncthreads();
  }
  n = n_l[0];
  if (row == 0) {
    c = c_l[0][col];
    const float p = n ? (float)(s_l[0][col] / n) : 0.0f;
    if (e < E) {
      counts[e] = c;
      probs[e] = p;
    }
    double share = e < E ? (double)c * p : 0.0;
#pragma unroll
    for (int m = kJoinCols / 2; m > 0; m >>= 1) share += __shfl_down(share, m, kJoinCols);
    if (col == 0) {
      __hip_atomic_store(&shares[blockIdx.x], share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             (int)gridDim.x - 1;
    }
  }
  __syncthreads();
  if (last && tid < 64) {
    double t = 0.0;
    for (int b = tid; b < (int)gridDim.x; b += 64)
      t += __hip_atomic_load(&shares[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) t += __shfl_down(t, m, 64);
    if (tid != 0) return;
    *loss = n ? (float)(t * E / ((double)n * K)) : 0.0f;
    *tokens = n;
    *status = n_l[1];
  }
}

// loss of counts and probs, by one workgroup
__device__ __forceinline__ void loss_of(int E, int K, int n, const int32_t* counts,
                                        const float* probs, double* part, float* loss) {
  const int tid = threadIdx.x, threads = blockDim.x;
  double s = 0.0;
  for (int e = tid; e < E; e += threads) s += (double)counts[e] * probs[e];
  part[tid] = s;
  __syncthreads();
  for (int m = threads >> 1; m > 0; m >>= 1) {
    if (tid < m) part[tid] += part[tid + m];
    __syncthreads();
  }
  if (tid == 0) *loss = n ? (float)(part[0] * E / ((double)n * K)) : 0.0f;
}
// Everything in one workgroup, for few rows.
template <bool BF16, int SLOTS>
__global__ __launch_bounds__(64 * kSmallWaves) void balance_small_kernel(
    BalanceArgs a, float* __restrict__ loss, int32_t* __restrict__ counts,
    float* __restrict__ probs, int32_t* __restrict__ tokens, int32_t* __restrict__ status) {
  extern __shared__ float lds[];
  __shared__ double part[64 * kSmallWaves];
  __shared__ int tally[2];
  float* red = lds;
  int* hist = reinterpret_cast<int*>(red + kSmallWaves * a.E);
  sum_rows<BF16, SLOTS, kSmallWaves>(a, 0, a.T, red, hist, tally);
  const int n = tally[0];
  for (int e = threadIdx.x; e < a.E; e += 64 * kSmallWaves) {
    double s = 0.0;
    for (int w = 0; w < kSmallWaves; ++w) s += red[w * a.E + e];
    counts[e] = hist[e];
    const float p = n ? (float)(s / n) : 0.0f;
    probs[e] = p;
    red[e] = p;  // (row 0: this thread's own)
  }
  __syncthreads();
  loss_of(a.E, a.K, n, hist, red, part, loss);
  if (threadIdx.x == 0) {
    *tokens = n;
    *status = tally[1];
  }
}

// The gradient, a wave per row.  (Stores that keep no place in the caches: T = 32768
// by 512 28.6 us instead of 32.9, but a sum over the gradient after it 6 us more.)
template <bool BF16, int SLOTS>
__global__ __launch_bounds__(64 * kWaves) void balance_vjp_kernel(
    BalanceArgs a, const int32_t* __restrict__ counts, const int32_t* __restrict__ tokens,
    const float* __restrict__ dloss, const float* __restrict__ dw, void* __restrict__ dz) {
  extern __shared__ float lds[];  // [waves, E]: the choices' gradients, else 0
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float* own = lds + wave * a.E;
  float f[SLOTS];  // dloss * E / N * counts / (N K)
  const int n = dloss ? *tokens : 0;
  const float scale =
      n > 0 ? (float)((double)*dloss * a.E / ((double)n * n * a.K)) : 0.0f;
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const int e = lane + 64 * j;
    f[j] = n > 0 && e < a.E ? scale * (float)counts[e] : 0.0f;
    if (dw && e < a.E) own[e] = 0.0f;
  }
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < a.T;
       t += (int64_t)gridDim.x * kWaves) {
    float v[SLOTS];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) v[j] = 0.0f;
    if (!a.mask || a.mask[t] != 0) {
      int ek = -1;
      float gk = 0.0f;
      bool first = false;
      if (dw) {
        // lane k: choice k's weight and gradient
        const bool mine = lane < a.K;
        const int64_t i = t * a.K + (mine ? lane : 0);
        const int e = a.idx[i];
        const bool in = mine && (uint32_t)e < (uint32_t)a.E;
        ek = in ? e : -1;
        const float zk = in ? logit<BF16>(a.z, t * a.ld + e) : -INFINITY;
        const float dk = in ? dw[i] : 0.0f;
        const float m = softmax_base(wave_max(zk));
        const float u = in ? __builtin_amdgcn_exp2f((zk - m) * kLog2e) : 0.0f;
        const float s = wave_add(u);
        const float w = s == 0.0f ? 0.0f : u / s;
        gk = w * (dk - wave_add(w * dk));
        // one expert chosen twice: its first lane takes the sum, in order
        first = in;
        float sum = 0.0f;
        for (int k = 0; k < a.K; ++k) {
          const int e2 = __builtin_amdgcn_readlane(ek, k);
          const float g2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(gk), k));
          if (e2 == ek) {
            sum += g2;
            if (k < lane) first = false;
          }
        }
        gk = sum;
      }
      if (dloss) {
        load_row<BF16, SLOTS>(a.z, a.ld, t, a.E, lane, v);
        softmax_row<SLOTS>(v);
        float d = 0.0f;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) d += v[j] * f[j];
        d = wave_add(d);
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) v[j] *= f[j] - d;
      }
      if (dw) {
        if (first) own[ek] = gk;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const int e = lane + 64 * j;
          if (e < a.E) v[j] += own[e];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (first) own[ek] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const int e = lane + 64 * j;
      if (e < a.E) {
        if constexpr (BF16)
          static_cast<uint16_t*>(dz)[t * a.E + e] = f32_to_bf16(v[j]);
        else
          static_cast<float*>(dz)[t * a.E + e] = v[j];
      }
    }
  }
}

// Rows a workgroup of the two-launch form: two per wave, more where that would
// make over 256 workgroups (one a CU; c4's 32768 rows 14.1 us and 6.0 for the
// second launch so, 13.5 and 6.8 with two a CU, 15.3 and 9.9 with four).
int part_rows(int64_t T) {
  return (int)std::max<int64_t>(2 * kPartWaves, (T + 255) / 256);
}
int part_groups(int64_t T) { return (int)((T + part_rows(T) - 1) / part_rows(T)); }
// One workgroup for everything: few rows
bool one_workgroup(int64_t T, int64_t E) { return T * ((E + 63) / 64) <= 256; }

struct BalanceScratch {
  int32_t* status;
  float* sums;
  int32_t *cnts, *tallies, *ticket;
  double* shares;
};
BalanceScratch carve_balance(Carve& c, int64_t T, int64_t E) {
  BalanceScratch b{};
  b.status = c.take<int32_t>(1);
  if (one_workgroup(T, E)) return b;
  const int64_t G = part_groups(T);
  b.sums = c.take<float>(G * E);
  b.cnts = c.take<int32_t>(G * E);
  b.tallies = c.take<int32_t>(2 * G);
  b.ticket = c.take<int32_t>(1);
  b.shares = c.take<double>((E + kJoinCols - 1) / kJoinCols);
  return b;
}

#define MLXR_BAL_SLOTS(CALL, BF)              \
  do {                                        \
    const int slots_ = (int)((E + 63) / 64);  \
    if (slots_ <= 1)                          \
      CALL(BF, 1);                            \
    else if (slots_ <= 2)                     \
      CALL(BF, 2);                            \
    else if (slots_ <= 4)                     \
      CALL(BF, 4);                            \
    else if (slots_ <= 8)                     \
      CALL(BF, 8);                            \
    else                                      \
      CALL(BF, 16);                           \
  } while (0)

}  // namespace

void plan_router_balance(Carve& c, int64_t T, int64_t E) { (void)carve_balance(c, T, E); }

hipError_t launch_router_balance(const void* z, bool bf16, int64_t ld, int64_t T, int64_t E,
                                 const int32_t* idx, int64_t K, const uint8_t* mask, float* loss,
                                 int32_t* counts, float* probs, int32_t* tokens, Carve ws,
                                 hipStream_t s) {
  const BalanceScratch b = carve_balance(ws, T, E);
  const BalanceArgs a{z, ld, T, (int)E, (int)K, idx, mask};
  ProfileScope prof("router_balance", s);
  if (one_workgroup(T, E)) {
    const size_t lds = (size_t)(kSmallWaves + 1) * E * 4;
#define MLXR_BAL_CALL(BF, S)                                             \
  balance_small_kernel<BF, S><<<1, 64 * kSmallWaves, lds, s>>>(a, loss, counts, probs, tokens, \
                                                               b.status)
    if (bf16)
      MLXR_BAL_SLOTS(MLXR_BAL_CALL, true);
    else
      MLXR_BAL_SLOTS(MLXR_BAL_CALL, false);
#undef MLXR_BAL_CALL
    return hipGetLastError();
  }
  const int G = part_groups(T), rows = part_rows(T);
  const size_t lds = ((size_t)(kPartWaves + 1) * E + 2) * 4;
#define MLXR_BAL_CALL(BF, S)                                                                 \
  balance_part_kernel<BF, S><<<G, 64 * kPartWaves, lds, s>>>(a, rows, b.sums, b.cnts, b.tallies, \
                                                             b.ticket)
  if (bf16)
    MLXR_BAL_SLOTS(MLXR_BAL_CALL, true);
  else
    MLXR_BAL_SLOTS(MLXR_BAL_CALL, false);
#undef MLXR_BAL_CALL
  balance_join_kernel<<<(unsigned)((E + kJoinCols - 1) / kJoinCols), kJoinCols * kJoinRows, 0,
                        s>>>(G, (int)E, (int)K, b.sums, b.cnts, b.tallies, b.shares, b.ticket,
                             loss, counts, probs, tokens, b.status);
  return hipGetLastError();
}

hipError_t launch_router_balance_vjp(const void* z, bool bf16, int64_t ld, int64_t T, int64_t E,
                                     const int32_t* idx, int64_t K, const uint8_t* mask,
                                     const int32_t* counts, const int32_t* tokens,
                                     const float* dloss, const float* dweights, void* dlogits,
                                     hipStream_t s) {
  if (T == 0) return hipSuccess;
  const BalanceArgs a{z, ld, T, (int)E, (int)K, idx, mask};
  ProfileScope prof("router_balance_vjp", s);
  const unsigned grid = (unsigned)std::min<int64_t>((T + kWaves - 1) / kWaves, 2048);
  const size_t lds = dweights ? (size_t)kWaves * E * 4 : 0;
#define MLXR_BAL_CALL(BF, S)                                                             \
  balance_vjp_kernel<BF, S><<<grid, 64 * kWaves, lds, s>>>(a, counts, tokens, dloss, dweights, \
                                                           dlogits)
  if (bf16)
    MLXR_BAL_SLOTS(MLXR_BAL_CALL, true);
  else
    MLXR_BAL_SLOTS(MLXR_BAL_CALL, false);
#undef MLXR_BAL_CALL
  return hipGetLastError();
}

}  // namespace mlxr_moe
