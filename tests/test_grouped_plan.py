"""The plan of grouped_mm_vjp's weight gradients: where the parts of every group lie, which
slice of the workspace a part is summed in and which slices are joined, whatever the offsets.

The kernel's own code is compiled for the host and made by one thread; what it writes is
checked against the arrays it is to stay in."""
import os
import subprocess
from pathlib import Path

import pytest
import torch

from test_grouped import BF16, F32, near, problem, to

gpu = pytest.mark.gpu
SRC = Path(__file__).resolve().parent.parent / "mlx-rs_amd" / "csrc"

PROGRAM = r"""
#include "grouped.hpp"
#include <cstdio>
#include <random>
#include <vector>
using namespace mlxr_moe;

struct OneThread {
  __host__ __device__ int tid() const { return 0; }
  __host__ __device__ int threads() const { return 1; }
  __host__ __device__ void sync() const {}
  template <class Op>
  __host__ __device__ int before(int, int*, Op) const { return 0; }
};

constexpr int32_t kStale = 0x7f7f7f7f;
static long bad = 0, joined = 0;
static void fail(const char* what, const std::vector<int32_t>& off, long R) {
  if (bad++ > 5) return;
  std::printf("%s: R %ld, offsets", what, R);
  for (size_t i = 0; i < off.size() && i < 12; ++i) std::printf(" %d", off[i]);
  std::printf("\n");
}

static void check(const std::vector<int32_t>& off, long R, long N, long K) {
  const int E = (int)off.size() - 1;
  GroupedArgs a{};
  a.offsets = off.data();
  a.R = R, a.E = E, a.C = (int32_t)N, a.J = (int32_t)K;
  a.chunk = (int32_t)grouped_chunk_rows(R, N, K);
  a.slices = (int32_t)grouped_slices(R, a.chunk);
  a = with_plan(a);
  const long words = plan_words(a.max_parts, a.slices);
  std::vector<int32_t> plan(words + 256, kStale);
  a.plan = plan.data();
  static int lds[kPlanWords];
  write_plan(a, OneThread{}, lds);
  for (long i = words; i < (long)plan.size(); ++i)
    if (plan[i] != kStale) return fail("written behind the plan", off, R);
  if (plan[0] != 0) return fail("first run", off, R);
  for (int x = 0; x < (int)kXcds; ++x)
    if (plan[x + 1] < plan[x] || plan[x + 1] - plan[x] > a.max_run)
      return fail("a run longer than its workgroups", off, R);
  const int parts = plan[kXcds];
  if (parts < E || parts > a.max_parts) return fail("parts", off, R);
  // the groups: offsets clamped, an entry below one before it as that one
  std::vector<long> tab(E + 1);
  long most = 0;
  for (int e = 0; e <= E; ++e) {
    const long o = off[e] < R ? off[e] : R;
    most = o > most ? o : most;
    tab[e] = most;
  }
  const int4* records = reinterpret_cast<const int4*>(plan.data() + kPlanHead);
  const int2* first = reinterpret_cast<const int2*>(plan.data() + kPlanHead + 4 * a.max_parts);
  int p = 0, slice = 0;
  for (int e = 0; e < E; ++e) {
    long at = tab[e];
    const int p0 = p, s0 = slice;
    bool several = false;
    do {
      if (p >= parts) return fail("a group without a part", off, R);
      const int4 r = records[p];
      if (r.x != e || r.y != at || r.z < 0 || r.z > a.chunk || r.y + r.z > tab[e + 1])
        return fail("a part's rows", off, R);
      if (r.w != -1 && (r.w != slice || r.w >= a.slices)) return fail("a part's slice", off, R);
      if (r.w >= 0) several = true, ++slice;
      at += r.z, ++p;
    } while (at < tab[e + 1]);
    if (several != (p - p0 > 1)) return fail("a slice of one part", off, R);
    for (int s = s0; s < slice; ++s)
      if (first[s].x != e || first[s].y != (s == s0 ? p - p0 : 0))
        return fail("a slice's group", off, R);
    joined += several;
  }
  if (p != parts) return fail("parts of no group", off, R);
  for (int s = slice; s < a.slices; ++s)
    if (first[s].x != 0 || first[s].y != 0) return fail("a slice of no group", off, R);
}

int main() {
  check({0, 16384, 0, 16384}, 16384, 64, 64);
  check({0, 16384, 0, 16384, 0, 16384}, 16384, 2048, 768);
  check({-5, 2147483647, 0, 70000, -2147483647}, 70000, 64, 64);
  check({0, 0}, 0, 64, 64);
  check({100, 5000}, 5000, 8, 8);
  std::mt19937 rng(1);
  const auto upto = [&](long n) { return (long)(rng() % (unsigned long)(n + 1)); };
  for (int i = 0; i < 4000; ++i) {
    const int E = 1 + (int)upto(i % 7 == 0 ? 1023 : 40);
    const long R = i % 5 == 0 ? 1L << upto(24) : upto(60000);
    const long N = 8 * (1 + upto(512)), K = 8 * (1 + upto(512));
    std::vector<int32_t> off(E + 1);
    for (auto& o : off) o = (int32_t)(upto(R + R / 8 + 20) - 10);
    if (i % 3 == 0) std::sort(off.begin(), off.end());           // as they should be
    if (i % 3 == 1) for (int e = 0; e <= E; ++e) off[e] = e & 1 ? (int32_t)R : 0;
    check(off, R, N, K);
  }
  std::printf("joined %ld bad %ld\n", joined, bad);
  return bad != 0 || joined < 1000;
}
"""


def test_plan_stays_in_its_arrays(tmp_path):
    (tmp_path / "plan.hip").write_text(PROGRAM)
    exe = tmp_path / "plan"
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "hip", "-O1", "-std=c++17",
                    "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-w", "-I", str(SRC), str(tmp_path / "plan.hip"), "-o",
                    str(exe)], check=True, capture_output=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


@gpu
@pytest.mark.parametrize("offsets", [[0, 16384, 0, 16384], [0, 9000, 7000, 12000, 3000, 16384],
                                     [500, 16384, 2 ** 31 - 1, -7, 16384], [0] * 30 + [16384]])
@pytest.mark.parametrize("need_dx", [False, True])
def test_weight_gradients_of_loose_offsets(pkg, dev, offsets, need_dx):
    """Offsets that do not ascend: dW as of the largest one up to each, and nothing behind it.
    Tolerance as in test_grouped.py."""
    R, K, N = 16384, 64, 40
    E = len(offsets) - 1
    x, _, dy, _, _ = problem(3, [R], K, N)
    w = torch.zeros((E, N, K), dtype=BF16)
    tab = torch.tensor(offsets).clamp(0, R).cummax(0).values
    o = torch.tensor(offsets, dtype=torch.int32)
    dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, o), dw_dtype=F32, need_dx=need_dx)
    for e in range(E):
        s = slice(int(tab[e]), int(tab[e + 1]))
        near(dw[e], dy[s].double().t() @ x[s].double(),
             dy[s].double().abs().t() @ x[s].double().abs(), s.stop - s.start + 1)
    # the C call with a workspace that holds garbage and guarded outputs
    lib, C = pkg._capi.lib(), pkg._capi
    n = lib.mlxr_moe_grouped_mm_vjp_workspace_size(R, E, N, K)
    ws = torch.full((n,), 0x7f, dtype=torch.uint8, device=dev)
    out = torch.full((E + 8, N, K), 7.0, device=dev)
    dyd, xd, wd, od = to(dev, dy, x, w, o)
    C.check(lib.mlxr_moe_grouped_mm_vjp(
        dyd.data_ptr(), xd.data_ptr(), R, K, wd.data_ptr(), E, N, od.data_ptr(), None, R, None,
        out[4:].data_ptr(), C.FLOAT32, ws.data_ptr(), n,
        torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[4:E + 4], dw)
    assert bool((out[:4] == 7).all()) and bool((out[E + 4:] == 7).all())
