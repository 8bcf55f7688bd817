"""grouped_mm, its gradients and grouped_qmm (products grouped by expert over ragged
groups of sorted rows) against plain 64-bit restatements.

Tolerances: products of bf16 values are exact in f32; a sum of n of them in f32 is off
by at most n * 2^-24 of the sum of their magnitudes (mass).  Storing rounds by 2^-8
(bf16) or 2^-24 (f32).  grouped_qmm's matrix instructions keep a product down to 2^-13
of the largest of the few products added at a time (up to 16 neighbouring ones are
counted): off by at most 16 * 2^-13 of each 16 products' largest.
"""
import pytest
import torch

from test_add_norm import decode8

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32, BF16 = torch.float32, torch.bfloat16


def problem(seed, counts, K, N, tail=0, mapped=None, spread=0.05):
    """x, w, dy, offsets, rows; `tail` rows behind the last group; mapped: rows of x."""
    g = torch.Generator().manual_seed(seed)
    E, R = len(counts), sum(counts) + tail
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(counts).cumsum(0)
    rows = None if mapped is None else torch.randint(0, mapped, (R,), generator=g,
                                                     dtype=torch.int32)
    x = torch.randn((R if mapped is None else mapped, K), generator=g).to(BF16)
    w = (torch.randn((E, N, K), generator=g) * spread).to(BF16)
    dy = torch.randn((R, N), generator=g).to(BF16)
    return x, w, dy, offsets, rows


def taken(x, rows):
    """The sorted rows of x in 64 bits, zeros for indices that name none."""
    x = x.double()
    if rows is None:
        return x
    ok = (rows >= 0) & (rows < x.shape[0])
    return torch.where(ok[:, None], x[torch.where(ok, rows, 0).long()], 0.0)


def forward64(xs, w, offsets):
    R, (E, N, K) = xs.shape[0], w.shape
    y = torch.zeros((R, N), dtype=torch.float64)
    mass = torch.zeros_like(y)
    for e in range(E):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        y[s] = xs[s] @ w[e].double().t()
        mass[s] = xs[s].abs() @ w[e].double().abs().t()
    return y, mass


def near(got, want, mass, n):
    tol = n * 2.0 ** -24 * mass
    tol = tol + HALF[got.dtype] * (want.abs() + tol) + 1e-38
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


# groups of rows: none, one, the tiles' edges, more than a tile, one expert alone
GROUPS = {
    "one": [1],
    "ones": [1, 0, 1, 1, 0, 0, 1, 1],
    "edges": [31, 32, 33, 0, 63, 64, 65, 1],
    "tall": [255, 0, 257, 256, 129],
    "skewed": [0, 700, 3, 0, 1],
    "none": [0, 0, 0],
    "many": [(7 * e) % 11 for e in range(300)],
    "few_of_many": [1 if e in (0, 77, 1023) else 0 for e in range(1024)],
    "16": [16, 17, 15, 8, 9, 7, 0, 2],
}
# K, N: whole tiles, odd ends
DIMS = [(64, 64), (512, 256), (8, 8), (200, 328), (1032, 424), (72, 264), (328, 72)]


@gpu
@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("K,N", DIMS)
@pytest.mark.parametrize("mapped", [None, 37])
def test_grouped_mm(pkg, dev, groups, K, N, mapped):
    if groups in ("many", "few_of_many") and K * N > 64 * 64:
        K, N = 72, 40
    counts = GROUPS[groups]
    x, w, _, offsets, rows = problem(K + N, counts, K, N, tail=5, mapped=mapped)
    out_dtype = F32 if K % 3 else BF16
    got = pkg.ops.grouped_mm(*to(dev, x, w, offsets, rows), out_dtype=out_dtype)
    y, mass = forward64(taken(x, rows), w, offsets)
    assert got.dtype == out_dtype
    near(got, y, mass, K)
    assert bool((got[sum(counts):] == 0).all())


@gpu
@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("K,N", DIMS)
@pytest.mark.parametrize("mapped", [None, 37])
def test_grouped_mm_vjp(pkg, dev, groups, K, N, mapped):
    if groups in ("many", "few_of_many") and K * N > 64 * 64:
        K, N = 72, 40
    counts = GROUPS[groups]
    x, w, dy, offsets, rows = problem(K * N, counts, K, N, tail=3, mapped=mapped)
    dw_dtype = BF16 if N % 3 else F32
    dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows), dw_dtype=dw_dtype)
    assert dx.dtype == BF16 and dw.dtype == dw_dtype
    # dx: the forward product of dy by the transposed weights
    want, mass = forward64(dy.double(), w.transpose(1, 2), offsets)
    near(dx, want, mass, N)
    xs, g = taken(x, rows), dy.double()
    want, mass = torch.zeros(w.shape, dtype=torch.float64), torch.zeros(w.shape,
                                                                        dtype=torch.float64)
    for e in range(len(counts)):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        want[e], mass[e] = g[s].t() @ xs[s], g[s].abs().t() @ xs[s].abs()
    near(dw, want, mass, max(counts) + 1)


@gpu
def test_grouped_mm_vjp_is_the_derivative(pkg, dev):
    """<dy, y(x + e u) - y(x - e u)> is 2 e <dx, u> (y is linear in x, and in w)."""
    x, w, dy, offsets, rows = problem(3, [5, 0, 70, 2], 72, 40, mapped=20)
    dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows), dw_dtype=F32)
    g = torch.Generator().manual_seed(1)
    u = torch.randn(x.shape, generator=g, dtype=torch.float64)
    v = torch.randn(w.shape, generator=g, dtype=torch.float64)
    for got, diff, m, half in (
            (dx.cpu().double() * u[rows.long()],
             [forward64(taken(x.double() + s * u, rows), w, offsets)[0] for s in (1, -1)], 40,
             2.0 ** -8),
            (dw.cpu().double() * v,
             [forward64(taken(x, rows), w.double() + s * v, offsets)[0] for s in (1, -1)], 77,
             2.0 ** -24)):
        want = (dy.double() * (diff[0] - diff[1])).sum() / 2
        scale = (dy.double().abs() * (diff[0] - diff[1]).abs()).sum() / 2 + got.abs().sum()
        assert abs(float(got.sum() - want)) <= (half + m * 2.0 ** -20) * float(scale)


@gpu
def test_rows_that_name_no_row_are_zeros(pkg, dev):
    x, w, dy, offsets, rows = problem(4, [40, 3, 300], 128, 64, mapped=9)
    rows[::7] = torch.tensor([-1, 9, 2 ** 31 - 1, -2 ** 31] * 20, dtype=torch.int32)[
        :len(rows[::7])]
    got = pkg.ops.grouped_mm(*to(dev, x, w, offsets, rows))
    assert bool((got[::7] == 0).all())
    y, mass = forward64(taken(x, rows), w, offsets)
    near(got, y, mass, 128)
    _, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows.long()), dw_dtype=F32,
                                   need_dx=False)
    xs = taken(x, rows)
    for e in range(3):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        near(dw[e], dy[s].double().t() @ xs[s], dy[s].double().abs().t() @ xs[s].abs(), 300)
    q, sc, _ = pkg.ops.quantize(x.to(dev), mode="mxfp8")
    wq, wsc, _ = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    got = pkg.ops.grouped_qmm(q, sc, wq, wsc, *to(dev, offsets, rows))
    assert bool((got[::7] == 0).all())


@gpu
def test_nan_and_inf_stay_in_their_rows(pkg, dev):
    x, w, dy, offsets, _ = problem(5, [33, 40, 2], 72, 40)
    x[3, 71], dy[34, 39], w[2, 5, 7] = torch.nan, torch.inf, torch.nan
    y = pkg.ops.grouped_mm(*to(dev, x, w, offsets)).cpu()
    bad = torch.isnan(y)
    assert bool(bad[3].all()) and bool(bad[73:, 5].all())
    bad[3], bad[73:, 5] = False, False
    assert not bool(bad.any())
    dx, dw = [t.cpu() for t in pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets))]
    off = ~torch.isfinite(dx)
    assert bool(off[34].all()) and bool(off[73:, 7].all())
    off[34], off[73:, 7] = False, False
    assert not bool(off.any())
    off = ~torch.isfinite(dw)
    assert bool(off[0, :, 71].all()) and bool(off[1, 39].all())
    off[0, :, 71], off[1, 39] = False, False
    assert not bool(off.any())


def values4(wq, sc):
    t = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    t = torch.cat([t, -t])
    v = torch.stack([t[(wq.long() >> (4 * i)) & 15] for i in range(8)], -1).flatten(-2)
    s = torch.ldexp(torch.ones_like(v), sc.long().repeat_interleave(32, -1) - 127)
    return v * s


def check_qmm(pkg, dev, q, sc, wq, wsc, offsets, rows, out_dtype, got=None):
    if got is None:
        got = pkg.ops.grouped_qmm(*to(dev, q, sc, wq, wsc, offsets, rows), out_dtype=out_dtype)
    assert got.dtype == out_dtype
    xs, w = taken(decode8(q, sc), rows), values4(wq, wsc)
    y, mass = forward64(xs, w, offsets)
    K = xs.shape[1]
    lost = torch.zeros_like(y)
    for e in range(w.shape[0]):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        if s.start == s.stop:
            continue
        for k in range(0, K, 16):
            lost[s] += (xs[s, None, k:k + 16].abs() * w[e][None, :, k:k + 16].abs()).amax(-1)
    tol = K * 2.0 ** -24 * mass + 16 * 2.0 ** -13 * lost
    tol = tol + HALF[out_dtype] * (y.abs() + tol) + 1e-38
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    return got


@gpu
@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("K,N", [(128, 64), (512, 256), (32, 8), (160, 104), (96, 264),
                                 (1056, 72), (2080, 40)])
@pytest.mark.parametrize("mapped", [None, 37])
def test_grouped_qmm(pkg, dev, groups, K, N, mapped):
    if groups in ("many", "few_of_many"):
        K, N = 96, 40
    counts = GROUPS[groups]
    x, w, _, offsets, rows = problem(K + N, counts, K, N, tail=5, mapped=mapped)
    # scales of every group their own
    x = x * torch.exp2(torch.randint(-6, 7, (x.shape[0], K // 32)).float()).repeat_interleave(
        32, -1)
    q, sc, _ = [t.cpu() if t is not None else t
                for t in pkg.ops.quantize(x.to(BF16).to(dev), mode="mxfp8")]
    wq, wsc, _ = [t.cpu() if t is not None else t
                  for t in pkg.ops.quantize(w.to(dev), mode="mxfp4")]
    got = check_qmm(pkg, dev, q, sc, wq, wsc, offsets, rows, F32 if K % 3 else BF16)
    assert bool((got[sum(counts):] == 0).all())


@gpu
def test_grouped_qmm_nan_scales(pkg, dev):
    x, w, _, offsets, _ = problem(6, [33, 2], 64, 40)
    x[3, 40] = torch.nan
    q, sc, _ = pkg.ops.quantize(x.to(dev), mode="mxfp8")
    w[1, 5, 7] = torch.inf
    wq, wsc, _ = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    bad = torch.isnan(pkg.ops.grouped_qmm(q, sc, wq, wsc, offsets.to(dev))).cpu()
    assert bool(bad[3].all()) and bool(bad[33:, 5].all())
    bad[3], bad[33:, 5] = False, False
    assert not bool(bad.any())


@gpu
def test_offsets_that_do_not_fit_stay_inside(pkg, dev):
    """Offsets past the rows are clamped; descending ones leave zeros or some group's rows."""
    x, w, dy, _, _ = problem(7, [64, 64], 64, 64)
    for off in ([0, 500, 900], [0, 100, 20], [0, -5, 128], [200, 300, 400], [0, 2 ** 31 - 1, 0]):
        o = torch.tensor(off, dtype=torch.int32)
        y = pkg.ops.grouped_mm(*to(dev, x, w, o))
        dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, o))
        assert y.shape == dx.shape == (128, 64) and dw.shape == w.shape
    o = torch.tensor([0, 100, 500], dtype=torch.int32)
    y = pkg.ops.grouped_mm(*to(dev, x, w, o))
    want, mass = forward64(x.double(), w, o.clamp_max(128))
    near(y, want, mass, 64)


@gpu
def test_no_rows(pkg, dev):
    x, w, dy, offsets, _ = problem(8, [0, 0], 64, 40)
    y = pkg.ops.grouped_mm(*to(dev, x, w, offsets))
    assert y.shape == (0, 40)
    dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets))
    assert dx.shape == (0, 64) and bool((dw == 0).all())
    rows = torch.zeros(0, dtype=torch.int32)
    xs = torch.ones((3, 64), dtype=BF16)
    assert pkg.ops.grouped_mm(*to(dev, xs, w, offsets, rows)).shape == (0, 40)


@gpu
def test_views_alignment_and_index_types(pkg, dev):
    x, w, dy, offsets, rows = problem(9, [20, 45], 64, 40, mapped=12)
    want = pkg.ops.grouped_mm(*to(dev, x, w, offsets, rows))
    wide = torch.zeros((12, 75), dtype=BF16, device=dev)
    wide[:, 5:69] = x.to(dev)
    flat = torch.zeros(w.numel() + 1, dtype=BF16, device=dev)
    flat[1:] = w.flatten().to(dev)  # off 16-byte alignment
    got = pkg.ops.grouped_mm(wide[:, 5:69].view(3, 4, 64), flat[1:].view(w.shape),
                             offsets.long().to(dev), rows.long().to(dev))
    assert torch.equal(got, want)
    a = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows))
    b = pkg.ops.grouped_mm_vjp(*to(dev, dy.t().contiguous().t(), x, w, offsets, rows))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dx, none = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows), need_dw=False)
    assert none is None and torch.equal(dx, a[0])
    none, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows), need_dx=False)
    assert none is None and torch.equal(dw, a[1])


@gpu
def test_on_a_stream_and_in_a_graph(pkg, dev):
    ops = pkg.ops
    x, w, dy, offsets, rows = to(dev, *problem(10, [300, 0, 10, 200], 256, 128, mapped=200))
    wq, wsc, _ = ops.quantize(w, mode="mxfp4")

    def step():
        q, sc, _ = ops.quantize(x, mode="mxfp8")
        return (ops.grouped_mm(x, w, offsets, rows), *ops.grouped_mm_vjp(dy, x, w, offsets, rows),
                ops.grouped_qmm(q, sc, wq, wsc, offsets, rows))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)).to(BF16))
        offsets[1:4] = 290 + k  # other groups, too
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------- refusals
def test_refusals(pkg):
    lib, C, err = pkg._capi.lib(), pkg._capi, pkg._capi.last_error

    def mm(x=16, x_rows=4, K=64, w=16, E=2, N=64, off=16, rows=None, R=4, out=16, dt=C.BFLOAT16):
        return lib.mlxr_moe_grouped_mm(x, x_rows, K, w, E, N, off, rows, R, out, dt, None)

    def vjp(dy=16, x=16, x_rows=4, K=64, w=16, E=2, N=64, off=16, rows=None, R=4, dx=16, dw=16,
            dt=C.BFLOAT16, ws=256, n=1 << 30):
        return lib.mlxr_moe_grouped_mm_vjp(dy, x, x_rows, K, w, E, N, off, rows, R, dx, dw, dt,
                                           ws, n, None)

    def qmm(x=16, xs=16, x_rows=4, K=64, w=16, ws=16, E=2, N=64, off=16, rows=None, R=4, out=16,
            dt=C.BFLOAT16):
        return lib.mlxr_moe_grouped_qmm(x, xs, x_rows, K, w, ws, E, N, off, rows, R, out, dt, None)

    shared = [(dict(R=-1), "bad shape"), (dict(K=0), "bad shape"), (dict(N=0), "bad shape"),
              (dict(E=0), "bad shape"), (dict(E=1025), "at most 1024"), (dict(N=60), "multiple"),
              (dict(K=60), "multiple"), (dict(K=1 << 17), "up to"),
              (dict(K=1 << 16, N=1 << 15), "under 2^30"), (dict(R=1 << 25, x_rows=1 << 25), "rows"),
              (dict(x_rows=5), "without rows' indices"),
              (dict(x_rows=1 << 30, rows=16), "under 4 GB"), (dict(off=None), "null"),
              (dict(off=18), "aligned"), (dict(rows=18), "aligned"), (dict(x=None), "null"),
              (dict(w=None), "null"), (dict(x=24), "aligned"), (dict(w=24), "aligned"),
              (dict(dt=2), "f32 or bf16")]
    for f in (mm, vjp, qmm):
        for kw, word in shared:
            assert f(**kw) == -1 and word in err(), (f, kw, err())
    for f in (mm, qmm):
        assert f(out=None) == -1 and "null" in err()
        assert f(out=24) == -1 and "aligned" in err()
        assert f(R=0, x_rows=0, x=None, out=None) == 0
    assert vjp(dx=None, dw=None) == -1 and "required" in err()
    assert vjp(dy=None) == -1 and "null" in err()
    assert vjp(dy=24) == -1 and "aligned" in err()
    assert vjp(dx=24) == -1 and "aligned" in err()
    assert vjp(dw=24) == -1 and "aligned" in err()
    assert qmm(xs=None) == -1 and "null" in err()
    assert qmm(ws=None) == -1 and "null" in err()
    assert qmm(xs=17) == -1 and "aligned" in err()
    assert qmm(K=40) == -1 and "multiple of 32" in err()


def test_python_refusals(pkg):
    ops, E = pkg.ops, pkg.MlxrMoeError
    x, w, dy, offsets, _ = problem(1, [2, 2], 64, 64)
    with pytest.raises(E, match="ROCm device"):
        ops.grouped_mm(x, w, offsets)
    with pytest.raises(E, match="ROCm device"):
        ops.grouped_mm_vjp(dy, x, w, offsets)


@gpu
def test_python_refusals_on_the_device(pkg, dev):
    ops, E = pkg.ops, pkg.MlxrMoeError
    x, w, dy, offsets, rows = to(dev, *problem(1, [2, 2], 64, 64, mapped=3))
    for bad, word in [((x, w, offsets[:2], rows), "offsets must be"),
                      ((x, w, offsets.float(), rows), "integer"),
                      ((x[:, :32], w, offsets, rows), "last dim"),
                      ((x, w, offsets, rows.view(2, 2)), "rows must be"),
                      ((x, w[0], offsets, rows), "w must be"),
                      ((x, w.float(), offsets, rows), "w must be"),
                      ((x.float(), w, offsets, rows), "x must be")]:
        with pytest.raises(E, match=word):
            ops.grouped_mm(*bad)
        with pytest.raises(E, match=word):
            ops.grouped_mm_vjp(dy, *bad)
    with pytest.raises(E, match="dy must be"):
        ops.grouped_mm_vjp(dy[:3], x, w, offsets, rows)
    with pytest.raises(E, match="unsupported dtype"):
        ops.grouped_mm(x, w, offsets, rows, out_dtype=torch.float16)
    q, sc, _ = ops.quantize(x, mode="mxfp8")
    wq, wsc, _ = ops.quantize(w, mode="mxfp4")
    with pytest.raises(E, match="last dim"):
        ops.grouped_qmm(q[:, :8], sc[:, :1], wq, wsc, offsets, rows)
    with pytest.raises(E, match="eight words"):
        ops.grouped_qmm(q, sc[:, :1], wq, wsc, offsets, rows)
    with pytest.raises(E, match="four words"):
        ops.grouped_qmm(q, sc, wq, wsc[..., :1], offsets, rows)


# Groups of few rows (the kernel that streams the weights): its 16-row parts' edges, many
# experts, inputs shorter and longer than a chunk, rows that name none.
FEW = {
    "one": [1],
    "eight": [0, 1, 1, 1, 0, 1, 1, 1, 1, 1] + [0] * 30,
    "edges": [15, 16, 17, 0, 1, 33] + [0] * 30,
    "spread": [(5 * e) % 4 for e in range(90)],
    "last": [0] * 511 + [40],
}


@gpu
@pytest.mark.parametrize("groups", sorted(FEW))
@pytest.mark.parametrize("K,N", [(8, 8), (264, 520), (512, 136), (2056, 24), (4104, 16)])
@pytest.mark.parametrize("mapped", [None, 37])
def test_few_rows(pkg, dev, groups, K, N, mapped):
    counts = FEW[groups]
    if len(counts) > 100:
        K, N = min(K, 520), min(N, 24)
    x, w, _, offsets, rows = problem(K + N, counts, K, N, tail=4, mapped=mapped)
    if mapped:
        rows[::5] = mapped
    out_dtype = BF16 if K % 3 else F32
    got = pkg.ops.grouped_mm(*to(dev, x, w, offsets, rows), out_dtype=out_dtype)
    near(got, *forward64(taken(x, rows), w, offsets), K)
    assert bool((got[sum(counts):] == 0).all())
    K = (K + 31) // 32 * 32
    x, w, _, offsets, rows = problem(K + N, counts, K, N, tail=4, mapped=mapped)
    if mapped:
        rows[::5] = -1
    q, sc, _ = [None if t is None else t.cpu()
                for t in pkg.ops.quantize((3 * x).to(dev), mode="mxfp8")]
    wq, wsc, _ = [None if t is None else t.cpu()
                  for t in pkg.ops.quantize(w.to(dev), mode="mxfp4")]
    got = check_qmm(pkg, dev, q, sc, wq, wsc, offsets, rows, out_dtype)
    assert bool((got[sum(counts):] == 0).all())


@gpu
@pytest.mark.parametrize("K,N,counts", [(72, 40, [3000, 0, 5, 1100]), (264, 520, [0, 2500]),
                                        (64, 64, [1024, 1025]), (8, 8, [20000]),
                                        (128, 136, [1] * 700 + [4000])])
def test_weight_gradients_of_long_groups(pkg, dev, K, N, counts):
    """Groups summed in several parts; the same bits at every call."""
    x, w, dy, offsets, rows = problem(sum(counts), counts, K, N, tail=9, mapped=500)
    args = to(dev, dy, x, w, offsets, rows)
    _, dw = pkg.ops.grouped_mm_vjp(*args, dw_dtype=F32, need_dx=False)
    xs, g = taken(x, rows), dy.double()
    for e in range(len(counts)):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        near(dw[e], g[s].t() @ xs[s], g[s].abs().t() @ xs[s].abs(), counts[e] + 1)
    _, half = pkg.ops.grouped_mm_vjp(*args, need_dx=False)
    assert torch.equal(half, dw.to(BF16))
    for _ in range(3):
        _, again = pkg.ops.grouped_mm_vjp(*args, dw_dtype=F32, need_dx=False)
        assert torch.equal(again, dw)


def test_workspace_refusals(pkg):
    lib, C, err = pkg._capi.lib(), pkg._capi, pkg._capi.last_error
    need = lib.mlxr_moe_grouped_mm_vjp_workspace_size(4096, 4, 64, 64)
    assert need > 0
    # (long groups need room for their parts)
    assert lib.mlxr_moe_grouped_mm_vjp_workspace_size(1 << 20, 4, 64, 64) > need

    def vjp(ws, n, dw=16):
        return lib.mlxr_moe_grouped_mm_vjp(16, 16, 4096, 64, 16, 4, 64, 16, None, 4096, None, dw,
                                           C.BFLOAT16, ws, n, None)

    assert vjp(256, need - 1) == -1 and "workspace too small" in err()
    assert vjp(None, need) == -1 and "workspace is NULL" in err()
    assert vjp(128, need) == -1 and "256-byte aligned" in err()


@gpu
def test_two_streams_at_once(pkg, dev):
    """Calls on two streams share nothing."""
    ops = pkg.ops
    sets = [to(dev, *problem(20 + i, [2000, 3, 0, 1500 + i], 136, 72, mapped=300))
            for i in range(2)]
    want = [(ops.grouped_mm(x, w, o, r), *ops.grouped_mm_vjp(dy, x, w, o, r))
            for x, w, dy, o, r in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, (x, w, dy, o, r) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append((ops.grouped_mm(x, w, o, r), *ops.grouped_mm_vjp(dy, x, w, o, r)))
    torch.cuda.synchronize()
    for outs, right in zip(got, want):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, right))


@gpu
def test_few_rows_with_nan_and_loose_offsets(pkg, dev):
    """The streaming kernel: what is not finite stays in its row and column; offsets that
    descend or pass the rows stay inside the arrays."""
    x, w, _, offsets, _ = problem(31, [1, 2, 0, 3] + [0] * 28, 264, 40)
    x[2, 263], w[3, 5, 7] = torch.nan, torch.inf
    bad = ~torch.isfinite(pkg.ops.grouped_mm(*to(dev, x, w, offsets)).cpu())
    assert bool(bad[2].all()) and bool(bad[3:, 5].all())
    bad[2], bad[3:, 5] = False, False
    assert not bool(bad.any())
    x, w, _, offsets, _ = problem(32, [1, 2, 0, 3] + [0] * 28, 160, 40)
    x[2, 159], w[3, 5, 7] = torch.nan, torch.nan
    q, sc, _ = pkg.ops.quantize(x.to(dev), mode="mxfp8")
    wq, wsc, _ = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    bad = torch.isnan(pkg.ops.grouped_qmm(q, sc, wq, wsc, offsets.to(dev))).cpu()
    assert bool(bad[2].all()) and bool(bad[3:, 5].all())
    bad[2], bad[3:, 5] = False, False
    assert not bool(bad.any())
    g = torch.Generator().manual_seed(33)
    for _ in range(4):
        o = torch.randint(-3, 12, (33,), generator=g, dtype=torch.int32).to(dev)
        assert pkg.ops.grouped_mm(x.to(dev), w.to(dev), o).shape == (6, 40)
        assert pkg.ops.grouped_qmm(q, sc, wq, wsc, o).shape == (6, 40)


@gpu
def test_arrays_past_32_bits(pkg, dev):
    """x, dy, dx and out of more than 2^32 bytes; rows at their ends."""
    ops, R, wide = pkg.ops, 66000, 32768
    g = torch.Generator(device=dev).manual_seed(40)
    big = torch.randint(-2, 3, (R, wide), generator=g, device=dev, dtype=torch.int8).to(BF16)
    w = torch.randint(-2, 3, (2, 8, wide), generator=g, device=dev, dtype=torch.int8).to(BF16)
    offsets = torch.tensor([0, 65000, R], dtype=torch.int32, device=dev)
    last = slice(R - 40, R)
    # (small whole numbers: every sum is exact in f32)
    y = ops.grouped_mm(big, w, offsets, out_dtype=F32)
    assert torch.equal(y[last], big[last].float() @ w[1].float().t())
    small = torch.randint(-2, 3, (R, 8), generator=g, device=dev, dtype=torch.int8).to(BF16)
    dx, dw = ops.grouped_mm_vjp(small, big, w, offsets, dw_dtype=F32)
    assert torch.equal(dx[last].float(), small[last].float() @ w[1].float())
    assert torch.equal(dw[1], small[65000:].float().t() @ big[65000:].float())
    del dx, dw, y
    wt = w.transpose(1, 2).contiguous()
    out = ops.grouped_mm(small, wt, offsets)
    assert torch.equal(out[last].float(), small[last].float() @ wt[1].float().t())
    del out
    dx, dw = ops.grouped_mm_vjp(big, small, wt, offsets, dw_dtype=F32)
    assert torch.equal(dx[last].float(), (big[last].float() @ wt[1].float()).to(BF16).float())
    assert torch.equal(dw[1], big[65000:].float().t() @ small[65000:].float())
