// C ABI of the products grouped by expert over sorted rows (declarations in
// include/mlxr_moe.h): every host-visible argument is checked, then kernels are
// enqueued on the caller's stream.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/mlxr_moe.h"
#include "grouped.hpp"
#include "nn.hpp"

using namespace mlxr_moe;

namespace {

int finish(const Status& st) { return st.ok ? 0 : capi_fail(st.what); }
hipStream_t as_stream(mlxr_moe_stream s) { return reinterpret_cast<hipStream_t>(s); }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool dtype_ok(int dt) { return dt == MLXR_MOE_FLOAT32 || dt == MLXR_MOE_BFLOAT16; }

// The shape that all of them share.  step: what N and K are multiples of; x_row: bytes
// of a row of x.
Status check_shape(const char* op, int64_t x_rows, int64_t K, int64_t E, int64_t N,
                   const int32_t* offsets, const int32_t* rows, int64_t R, int64_t k_step,
                   int64_t x_row) {
  const std::string o(op);
  if (R < 0 || x_rows < 0 || K <= 0 || N <= 0 || E <= 0) return Status::error(o + ": bad shape");
  if (E > kMaxExperts)
    return Status::error(o + ": at most " + std::to_string(kMaxExperts) + " experts");
  if (K % k_step || N % 8)
    return Status::error(o + ": K must be a multiple of " + std::to_string(k_step) +
                         " and N of 8, got " + std::to_string(K) + " and " + std::to_string(N));
  if (K > kMaxGroupedDims || N > kMaxGroupedDims)
    return Status::error(o + ": K and N up to " + std::to_string(kMaxGroupedDims));
  if (N * K >= ((int64_t)1 << 30))
    return Status::error(o + ": one expert's weights must be under 2^30 values");
  if (R > kMaxGroupedRows || !grouped_grid_ok(R, E, N > K ? N : K))
    return Status::error(o + ": too many rows");
  if (!rows && R && x_rows != R)
    return Status::error(o + ": x has " + std::to_string(x_rows) + " rows, " +
                         std::to_string(R) + " without rows' indices");
  if (rows && x_rows * x_row >= ((int64_t)1 << 32) - (1 << 20))
    return Status::error(o + ": x must be under 4 GB where rows' indices are given");
  if (!offsets) return Status::error(o + ": null array");
  if (!aligned(offsets, 4) || !aligned(rows, 4))
    return Status::error(o + ": offsets and rows must be aligned to their elements");
  return Status{};
}

// dW's plan, and the parts of groups that are summed in several.
struct VjpScratch {
  int32_t* plan;
  float* parts;
};
VjpScratch plan_vjp(Carve& c, int64_t R, int64_t E, int64_t N, int64_t K) {
  const int64_t chunk = grouped_chunk_rows(R, N, K), slices = grouped_slices(R, chunk);
  VjpScratch v;
  v.plan = c.take<int32_t>(plan_words(grouped_chunks(R, E, chunk), slices));
  v.parts = c.take<float>(slices * N * K);
  return v;
}

}  // namespace

extern "C" {

int mlxr_moe_grouped_mm(const void* x, int64_t x_rows, int64_t K, const void* w, int64_t E,
                        int64_t N, const int32_t* offsets, const int32_t* rows, int64_t R,
                        void* out, int out_dtype, mlxr_moe_stream stream) {
  const Status st = check_shape("grouped_mm", x_rows, K, E, N, offsets, rows, R, 8, 2 * K);
  if (!st.ok) return finish(st);
  if (!dtype_ok(out_dtype)) return capi_fail("grouped_mm: out must be f32 or bf16");
  if (!w || (R && ((!x && x_rows) || !out))) return capi_fail("grouped_mm: null array");
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(out, 16))
    return capi_fail("grouped_mm: x, w and out must be 16-byte aligned");
  if (!R) return 0;
  GroupedArgs a{};
  a.m = x, a.j = w, a.offsets = offsets, a.rows = rows, a.out = out;
  a.R = R, a.x_rows = x_rows, a.E = (int32_t)E, a.J = (int32_t)N, a.C = (int32_t)K;
  a.out_f32 = out_dtype == MLXR_MOE_FLOAT32;
  ProfileScope prof("grouped_mm", as_stream(stream));
  return finish(from_hip(launch_grouped_mm(a, as_stream(stream)), "grouped_mm"));
}

size_t mlxr_moe_grouped_mm_vjp_workspace_size(int64_t R, int64_t E, int64_t N, int64_t K) {
  Carve c(nullptr);
  if (R >= 0 && E > 0 && N > 0 && K > 0) plan_vjp(c, R, E, N, K);
  return c.off;
}

int mlxr_moe_grouped_mm_vjp(const void* dy, const void* x, int64_t x_rows, int64_t K,
                            const void* w, int64_t E, int64_t N, const int32_t* offsets,
                            const int32_t* rows, int64_t R, void* dx, void* dw, int dw_dtype,
                            void* workspace, size_t workspace_size, mlxr_moe_stream stream) {
  Status st = check_shape("grouped_mm_vjp", x_rows, K, E, N, offsets, rows, R, 8, 2 * K);
  if (!st.ok) return finish(st);
  if (!dtype_ok(dw_dtype)) return capi_fail("grouped_mm_vjp: dw must be f32 or bf16");
  if (!dx && !dw) return capi_fail("grouped_mm_vjp: dx or dw is required");
  if ((R && !dy) || (dx && !w) || (dw && x_rows && !x))
    return capi_fail("grouped_mm_vjp: null array");
  if (!aligned(dy, 16) || !aligned(x, 16) || !aligned(w, 16) || !aligned(dx, 16) ||
      !aligned(dw, 16))
    return capi_fail("grouped_mm_vjp: arrays must be 16-byte aligned");
  Carve plan(nullptr);
  plan_vjp(plan, R, E, N, K);
  if (dw) {
    if (plan.off > workspace_size)
      return capi_fail("grouped_mm_vjp: workspace too small: need " + std::to_string(plan.off) +
                       " bytes, got " + std::to_string(workspace_size));
    if (!workspace) return capi_fail("grouped_mm_vjp: workspace is NULL");
    if (!aligned(workspace, 256))
      return capi_fail("grouped_mm_vjp: workspace must be 256-byte aligned");
  }
  hipStream_t s = as_stream(stream);
  GroupedArgs g{};  // dW
  if (dw) {
    g.m = dy, g.j = x, g.offsets = offsets, g.rows = rows, g.out = dw;
    g.R = R, g.x_rows = x_rows, g.E = (int32_t)E, g.J = (int32_t)K, g.C = (int32_t)N;
    g.out_f32 = dw_dtype == MLXR_MOE_FLOAT32;
    Carve c(workspace);
    const VjpScratch v = plan_vjp(c, R, E, N, K);
    g.plan = v.plan, g.parts = v.parts;
    g.chunk = (int32_t)grouped_chunk_rows(R, N, K);
    g.slices = (int32_t)grouped_slices(R, g.chunk);
  }
  const bool both = dx && R && dw;
  if (dx && R) {
    GroupedArgs a{};
    a.m = dy, a.j = w, a.offsets = offsets, a.out = dx;
    a.R = R, a.x_rows = R, a.E = (int32_t)E, a.J = (int32_t)K, a.C = (int32_t)N;
    ProfileScope prof("grouped_dx", s);
    st = from_hip(launch_grouped_dx(a, both ? &g : nullptr, s), "grouped_mm_vjp dx");
    if (!st.ok) return finish(st);
  }
  if (dw) {
    ProfileScope prof("grouped_dw", s);
    st = from_hip(launch_grouped_dw(g, both, s), "grouped_mm_vjp dw");
  }
  return finish(st);
}

int mlxr_moe_grouped_qmm(const uint32_t* x, const uint8_t* x_scales, int64_t x_rows, int64_t K,
                         const uint32_t* w, const uint8_t* w_scales, int64_t E, int64_t N,
                         const int32_t* offsets, const int32_t* rows, int64_t R, void* out,
                         int out_dtype, mlxr_moe_stream stream) {
  const Status st = check_shape("grouped_qmm", x_rows, K, E, N, offsets, rows, R, 32, K);
  if (!st.ok) return finish(st);
  if (!dtype_ok(out_dtype)) return capi_fail("grouped_qmm: out must be f32 or bf16");
  if (!w || !w_scales || (R && (((!x || !x_scales) && x_rows) || !out)))
    return capi_fail("grouped_qmm: null array");
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(out, 16) || !aligned(x_scales, 4) ||
      !aligned(w_scales, 4))
    return capi_fail("grouped_qmm: x, w and out must be 16-byte aligned, the scales 4-byte");
  if (!R) return 0;
  GroupedArgs a{};
  a.m = x, a.j = w, a.ms = x_scales, a.js = w_scales, a.offsets = offsets, a.rows = rows;
  a.out = out;
  a.R = R, a.x_rows = x_rows, a.E = (int32_t)E, a.J = (int32_t)N, a.C = (int32_t)K;
  a.out_f32 = out_dtype == MLXR_MOE_FLOAT32;
  ProfileScope prof("grouped_qmm", as_stream(stream));
  return finish(from_hip(launch_grouped_qmm(a, as_stream(stream)), "grouped_qmm"));
}

}  // extern "C"
