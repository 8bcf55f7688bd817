"""Rows that belong to no group, and rows whose index names no row of x: zeros, whatever the
operands hold.  Kernels of every size take part: outputs are given full of sevens to the C
calls, so that what is not written shows.  Tolerances as in test_grouped.py."""
import pytest
import torch

from test_grouped import BF16, F32, forward64, near, problem, taken, to

gpu = pytest.mark.gpu


class Filled:
    """The C calls into outputs that hold sevens."""

    def __init__(self, pkg, dev):
        self.lib, self.C, self.dev = pkg._capi.lib(), pkg._capi, dev

    def call(self, name, *args):
        args = [t.data_ptr() if isinstance(t, torch.Tensor) else t for t in args]
        self.C.check(getattr(self.lib, f"mlxr_moe_{name}")(
            *args, torch.cuda.current_stream().cuda_stream))

    def mm(self, x, w, offsets, rows, R):
        E, N, K = w.shape
        out = torch.full((R, N), 7.0, dtype=F32, device=self.dev)
        self.call("grouped_mm", x, x.shape[0], K, w, E, N, offsets, rows, R, out, self.C.FLOAT32)
        return out

    def vjp(self, dy, x, w, offsets, rows):
        E, N, K = w.shape
        R = dy.shape[0]
        dx = torch.full((R, K), 7.0, dtype=BF16, device=self.dev)
        dw = torch.full((E, N, K), 7.0, dtype=F32, device=self.dev)
        n = self.lib.mlxr_moe_grouped_mm_vjp_workspace_size(R, E, N, K)
        ws = torch.empty(n, dtype=torch.uint8, device=self.dev)
        self.call("grouped_mm_vjp", dy, x, x.shape[0], K, w, E, N, offsets, rows, R, dx, dw,
                  self.C.FLOAT32, ws, n)
        return dx, dw

    def qmm(self, x, xs, w, ws, offsets, rows, R):
        E, N, K = w.shape[0], w.shape[1], w.shape[2] * 8
        out = torch.full((R, N), 7.0, dtype=F32, device=self.dev)
        self.call("grouped_qmm", x, xs, x.shape[0], K, w, ws, E, N, offsets, rows, R, out,
                  self.C.FLOAT32)
        return out


# groups: one token's (the streaming kernels), the small tiles, the large ones (of 10 groups,
# enough columns for 256 of them)
CASES = {
    "stream": ([1, 0, 2, 1] + [0] * 28, 96, 40),
    "small": ([70, 0, 33, 200], 96, 40),
    "one": ([64], 64, 64),
    "large": ([129, 255, 300, 0, 600, 128, 1, 257, 400, 140], 64, 4096),
}


def shifted(case, before, after, seed, mapped=None):
    """A problem of which the first `before` and the last `after` rows are no group's."""
    counts, K, N = CASES[case]
    x, w, dy, offsets, rows = problem(seed, counts, K, N, tail=before + after, mapped=mapped)
    return x, w, dy, offsets + before, rows


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
@pytest.mark.parametrize("before,after", [(1, 0), (5, 3), (150, 0)])
@pytest.mark.parametrize("mapped", [None, 37])
def test_rows_before_the_first_group_are_zeros(pkg, dev, case, before, after, mapped):
    x, w, dy, offsets, rows = shifted(case, before, after, before, mapped)
    R, K, used = dy.shape[0], w.shape[2], slice(before, dy.shape[0] - after)
    c = Filled(pkg, dev)
    xd, wd, dyd, od, rd = to(dev, x, w, dy, offsets, rows)

    def outside(y):
        return bool((y[:used.start] == 0).all()) and bool((y[used.stop:] == 0).all())

    y = c.mm(xd, wd, od, rd, R)
    assert outside(y)
    near(y, *forward64(taken(x, rows), w, offsets), K)
    q, sc, _ = pkg.ops.quantize(xd, mode="mxfp8")
    wq, wsc, _ = pkg.ops.quantize(wd, mode="mxfp4")
    y = c.qmm(q, sc, wq, wsc, od, rd, R)
    assert outside(y) and bool((y[used] != 7).all())
    dx, dw = c.vjp(dyd, xd, wd, od, rd)
    assert outside(dx)
    near(dx, *forward64(dy.double(), w.transpose(1, 2), offsets), w.shape[1])
    xs, g = taken(x, rows), dy.double()
    for e in range(w.shape[0]):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        near(dw[e], g[s].t() @ xs[s], g[s].abs().t() @ xs[s].abs(), s.stop - s.start + 1)


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
def test_a_slice_of_the_offsets(pkg, dev, case):
    """The experts of one rank over all rows: those of the others' come out as zeros."""
    x, w, _, offsets, _ = problem(2, CASES[case][0], *CASES[case][1:])
    E = w.shape[0]
    a, b = E // 4, max(E * 3 // 4, 1)
    want = pkg.ops.grouped_mm(*to(dev, x, w, offsets))
    junk = torch.full_like(want, 7.0)
    del junk  # (what an unwritten output would hold)
    got = pkg.ops.grouped_mm(*to(dev, x, w[a:b], offsets[a:b + 1]))
    s = slice(int(offsets[a]), int(offsets[b]))
    assert bool((got[:s.start] == 0).all()) and bool((got[s.stop:] == 0).all())
    near(got, *forward64(x.double(), w[a:b], offsets[a:b + 1]), w.shape[2])


NONE = torch.tensor([-1, 37, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)


def padded(case, seed):
    """A problem over 37 rows of x in which every seventh sorted row names none."""
    x, w, dy, offsets, rows = shifted(case, 2, 3, seed, mapped=37)
    bad = torch.zeros(rows.numel(), dtype=torch.bool)
    bad[1::7] = True
    bad[2], bad[-4] = True, True  # the first and the last group's ends
    rows[bad] = NONE.repeat(rows.numel())[: int(bad.sum())]
    return x, w, dy, offsets, rows, bad


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
def test_rows_that_name_none_are_zeros_by_any_weights(pkg, dev, case):
    """Infinities and NaN in the weights reach the rows of their group that name a row of x, and
    no other."""
    x, w, _, offsets, rows, bad = padded(case, 11)
    w[0, 3, 5], w[-1, 7, 0], w[0, 8] = torch.nan, torch.inf, -torch.inf
    c, R = Filled(pkg, dev), rows.numel()
    xd, wd, od, rd = to(dev, x, w, offsets, rows)
    y = c.mm(xd, wd, od, rd, R).cpu()
    assert bool((y[bad] == 0).all())
    ok = ~bad
    ok[: int(offsets[0])], ok[int(offsets[-1]):] = False, False
    last = slice(int(offsets[-2]), int(offsets[-1]))
    assert not bool(torch.isfinite(y[last, 7][ok[last]]).any())
    assert bool(torch.isfinite(y[:, 10]).all())
    q, sc, _ = pkg.ops.quantize(xd, mode="mxfp8")
    wq, wsc, _ = pkg.ops.quantize(wd, mode="mxfp4")  # (scale bytes of 255)
    assert bool((wsc == 255).any())
    y = c.qmm(q, sc, wq, wsc, od, rd, R).cpu()
    assert bool((y[bad] == 0).all())
    assert bool(torch.isnan(y[last, 7][ok[last]]).all())
    assert bool(torch.isfinite(y[:, 10]).all())


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
@pytest.mark.parametrize("long", [False, True])
def test_rows_that_name_none_add_nothing(pkg, dev, case, long):
    """dW of rows that name none, whatever their dy: the same bits as with zeros there."""
    x, w, dy, offsets, rows, bad = padded(case, 12)
    if long:  # one group, several parts of its rows and several tables of their indices
        n = 3000
        g = torch.Generator().manual_seed(4)
        offsets = torch.tensor([0, n], dtype=torch.int32)
        dy = torch.randn((n, w.shape[1]), generator=g).to(BF16)
        rows = torch.randint(-9, 46, (n,), generator=g, dtype=torch.int32)
        bad = (rows < 0) | (rows >= 37)
        w = w[:1]
    clean = torch.where(bad[:, None], 0.0, dy.float()).to(BF16)
    dirty = dy.clone()
    dirty[bad] = torch.tensor([torch.nan, torch.inf, -torch.inf, 3e38])[
        torch.arange(int(bad.sum())) % 4][:, None].to(BF16)
    c = Filled(pkg, dev)
    a = c.vjp(*to(dev, clean, x, w, offsets, rows))[1]
    b = c.vjp(*to(dev, dirty, x, w, offsets, rows))[1]
    assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
    xs, g = taken(x, rows), clean.double()
    for e in range(w.shape[0]):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        near(a[e], g[s].t() @ xs[s], g[s].abs().t() @ xs[s].abs(), s.stop - s.start + 1)
