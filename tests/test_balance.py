"""router_balance (the load-balance loss with its counts) and its gradient,
against plain 64-bit restatements of their formulas.

Tolerances: a probability is exp2 of (z - max) log2(e), rounded twice, over the
sum of such: off by (|z - max| + 4) * 2^-22 of itself at most for each of the
two, so by 2 (R + 4) 2^-22 with R the range of the logits.  Sums of n
non-negative terms in f32 add n * 2^-24 of themselves.
"""
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu


def inputs(seed, T, E, K, dtype=torch.float32, mask=None, distinct=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((T, E), generator=g) * 1.5).to(dtype)
    if distinct:
        idx = torch.rand((T, E), generator=g).topk(K, dim=1).indices.to(torch.int32)
    else:
        idx = torch.randint(0, E, (T, K), generator=g, dtype=torch.int32)
    m = None
    if mask == "some":
        m = torch.rand(T, generator=g) < 0.7
    elif mask == "none":
        m = torch.zeros(T, dtype=torch.bool)
    elif mask == "one":
        m = torch.arange(T) == T // 2
    return z, idx, m


def probs64(z):
    z = z.double()
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top))
    s = p.sum(1, keepdim=True)
    return torch.where(s == 0, torch.zeros_like(p), p / torch.where(s == 0, 1.0, s))


def forward64(z, idx, mask):
    T, E = z.shape
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.bool()
    n = int(keep.sum())
    i = idx.long()[keep].reshape(-1)
    counts = torch.bincount(i[(i >= 0) & (i < E)], minlength=E)
    probs = probs64(z[keep]).sum(0) / max(n, 1)
    loss = E * (counts.double() * probs).sum() / max(n * idx.shape[1], 1)
    return loss, counts, probs, n


def vjp64(z, idx, mask, dloss, dw):
    """By formula, term by term; and each element's magnitude of terms."""
    T, E = z.shape
    K = idx.shape[1]
    _, counts, _, n = forward64(z, idx, mask)
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.bool()
    out = torch.zeros((T, E), dtype=torch.float64)
    mass = torch.zeros_like(out)
    if dloss is not None and n:
        p, f = probs64(z), counts.double() / (n * K)
        d = (p * f).sum(1, keepdim=True)
        out += dloss * E / n * p * (f - d)
        mass += abs(dloss) * E / n * p * (f + d)
    if dw is not None:
        for t in range(T):
            ok = [(k, int(e)) for k, e in enumerate(idx[t].tolist()) if 0 <= e < E]
            if not ok:
                continue
            w = probs64(z[t, [e for _, e in ok]][None])[0]
            g = dw[t, [k for k, _ in ok]].double()
            inner = (w * g).sum()
            for j, (_, e) in enumerate(ok):
                out[t, e] += w[j] * (g[j] - inner)
                mass[t, e] += w[j] * (g[j].abs() + (w * g.abs()).sum())
    return out * keep[:, None], mass * keep[:, None]


def rel_p(z, mask):
    """The bound on a probability's relative error, over the counted rows."""
    v = z if mask is None else z[mask.bool()]
    v = v[torch.isfinite(v)].double()
    r = float(v.max() - v.min()) if v.numel() else 0.0
    return 2 * (r + 4) * 2.0 ** -22


def check_forward(ops, dev, z, idx, mask):
    loss, counts, probs, tokens = ops.router_balance(
        z.to(dev), idx.to(dev), None if mask is None else mask.to(dev))
    want, c, p, n = forward64(z, idx, mask)
    assert torch.equal(counts.cpu().long(), c)
    assert int(tokens) == n
    tol = rel_p(z, mask) + z.shape[0] * 2.0 ** -24 + 2.0 ** -23
    assert bool(((probs.cpu().double() - p).abs() <= tol * p).all())
    assert abs(float(loss) - float(want)) <= tol * abs(float(want))
    return loss, counts, probs, tokens


def check_vjp(ops, dev, z, idx, mask, counts, tokens, dloss, dw):
    got = ops.router_balance_vjp(
        z.to(dev), idx.to(dev), counts, tokens,
        None if dloss is None else torch.tensor(dloss, device=dev),
        None if mask is None else mask.to(dev), None if dw is None else dw.to(dev))
    assert got.dtype == z.dtype and got.shape == z.shape
    want, mass = vjp64(z, idx, mask, dloss, dw)
    # two probabilities in each term, and sums of E and K terms
    n = z.shape[1] + idx.shape[1]
    tol = (3 * rel_p(z, mask) + (n + 8) * 2.0 ** -23) * mass
    if z.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol + 1e-38).all()), float((err - tol).max())
    return got


# ------------------------------------------------------------------ refusals
def test_refusals(pkg):
    lib, C = pkg._capi.lib(), pkg._capi

    def fwd(z=16, dt=C.FLOAT32, ld=8, T=4, E=8, idx=16, K=2, loss=16, ws=None, n=0):
        return lib.mlxr_moe_router_balance(z, dt, ld, T, E, idx, K, None, loss, 16, 16, 16, ws, n,
                                           None)

    assert fwd(dt=C.UINT8) == -1 and "f32 or bf16" in C.last_error()
    assert fwd(ld=7) == -1 and "bad shape" in C.last_error()
    assert fwd(T=-1) == -1 and "bad shape" in C.last_error()
    assert fwd(E=1025, ld=1025) == -1 and "at most 1024" in C.last_error()
    assert fwd(K=0) == -1 and "k must be" in C.last_error()
    assert fwd(K=65) == -1 and "k must be" in C.last_error()
    assert fwd(T=2 ** 31) == -1 and "too many" in C.last_error()
    assert fwd(z=None) == -1 and "null array" in C.last_error()
    assert fwd(idx=None) == -1 and "null array" in C.last_error()
    assert fwd(loss=None) == -1 and "null array" in C.last_error()
    assert fwd(z=18) == -1 and "aligned" in C.last_error()
    assert fwd() == -1 and "workspace" in C.last_error()
    assert fwd(ws=8, n=1 << 20) == -1 and "256-byte" in C.last_error()

    def bwd(dloss=16, dw=None, counts=16, tokens=16, dz=16, K=2):
        return lib.mlxr_moe_router_balance_vjp(16, C.FLOAT32, 8, 4, 8, 16, K, None, counts,
                                               tokens, dloss, dw, dz, None)

    assert bwd(dloss=None) == -1 and "required" in C.last_error()
    assert bwd(counts=None) == -1 and "counts and tokens" in C.last_error()
    assert bwd(dz=None) == -1 and "null array" in C.last_error()
    assert bwd(dz=18) == -1 and "aligned" in C.last_error()
    assert bwd(K=65) == -1 and "k must be" in C.last_error()
    assert lib.mlxr_moe_router_balance_vjp(None, C.FLOAT32, 8, 0, 8, None, 2, None, None, None,
                                           None, 16, None, None) == 0  # no tokens
    big = lib.mlxr_moe_router_balance_workspace_size(100000, 512)
    assert 0 < big < 1 << 23


def test_python_refusals(pkg):
    ops, Err = pkg.ops, pkg.MlxrMoeError
    z, idx = torch.zeros(4, 8), torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(Err, match="ROCm device"):
        ops.router_balance(z, idx)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


@gpu
def test_python_refusals_on_device(pkg, dev):
    ops, Err = pkg.ops, pkg.MlxrMoeError
    z, idx = torch.zeros(4, 8, device=dev), torch.zeros((4, 2), dtype=torch.int32, device=dev)
    with pytest.raises(Err, match="over logits"):
        ops.router_balance(z, idx[:3])
    with pytest.raises(Err, match="mask must be bool"):
        ops.router_balance(z, idx, torch.ones(4, device=dev))
    with pytest.raises(Err, match="one value per token"):
        ops.router_balance(z, idx, torch.ones(3, dtype=torch.bool, device=dev))
    with pytest.raises(Err, match="unsupported dtype"):
        ops.router_balance(z.half(), idx)
    with pytest.raises(Err, match="integer"):
        ops.router_balance(z, idx.float())
    _, counts, _, tokens = ops.router_balance(z, idx)
    one = torch.ones((), device=dev)
    with pytest.raises(Err, match="required"):
        ops.router_balance_vjp(z, idx)
    with pytest.raises(Err, match="counts and tokens"):
        ops.router_balance_vjp(z, idx, dloss=one)
    with pytest.raises(Err, match="one float32"):
        ops.router_balance_vjp(z, idx, counts, tokens, one.double())
    with pytest.raises(Err, match="counts must be int32"):
        ops.router_balance_vjp(z, idx, counts[:4], tokens, one)
    with pytest.raises(Err, match="must match"):
        ops.router_balance_vjp(z, idx, counts, tokens, one, None, torch.zeros(4, 3, device=dev))


# ------------------------------------------------------------------- results
SIZES = [(1, 2, 1), (1, 128, 8), (2, 3, 3), (7, 60, 4), (64, 128, 8), (65, 64, 64), (300, 65, 2),
         (128, 223, 10), (1000, 128, 8), (1037, 512, 10), (333, 1000, 6), (2000, 1024, 1),
         (20000, 16, 2)]


@gpu
@pytest.mark.parametrize("T,E,K", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [None, "some"])
def test_forward_and_gradient(pkg, dev, T, E, K, dtype, mask):
    z, idx, m = inputs(T + E, T, E, K, dtype, mask)
    _, counts, _, tokens = check_forward(pkg.ops, dev, z, idx, m)
    rows = slice(0, min(T, 400))  # the weights' term is checked row by row
    g = torch.Generator().manual_seed(T)
    check_vjp(pkg.ops, dev, z, idx, m, counts, tokens, -0.7, None)
    dw = torch.randn((T, K), generator=g)
    got = pkg.ops.router_balance_vjp(z.to(dev), idx.to(dev), None, None, None,
                                     None if m is None else m.to(dev), dw.to(dev))
    want, mass = vjp64(z[rows], idx[rows], None if m is None else m[rows], None, dw[rows])
    tol = (3 * rel_p(z, m) + (K + 8) * 2.0 ** -23) * mass
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((got.cpu().double()[rows] - want).abs() <= tol + 1e-38).all())


@gpu
@pytest.mark.parametrize("T", [5, 700])
def test_both_terms_and_repeated_choices(pkg, dev, T):
    """An expert chosen twice or more in a row: counted each time, its
    gradient the sum of its choices' terms."""
    z, idx, m = inputs(T, T, 24, 6, mask="some", distinct=False)
    idx[0] = 7
    _, counts, _, tokens = check_forward(pkg.ops, dev, z, idx, m)
    dw = torch.randn((T, 6), generator=torch.Generator().manual_seed(1))
    check_vjp(pkg.ops, dev, z, idx, m, counts, tokens, 0.3, dw)


@gpu
@pytest.mark.parametrize("T", [6, 900])
@pytest.mark.parametrize("mask", ["none", "one"])
def test_masks_that_leave_little(pkg, dev, T, mask):
    z, idx, m = inputs(T, T, 40, 3, mask=mask)
    loss, counts, probs, tokens = check_forward(pkg.ops, dev, z, idx, m)
    if mask == "none":
        assert float(loss) == 0.0 and float(probs.abs().max()) == 0.0
    dw = torch.ones((T, 3))
    got = check_vjp(pkg.ops, dev, z, idx, m, counts, tokens, 1.0, dw)
    assert bool((got.cpu()[~m] == 0).all())
    # a masked row's logits do not matter, whatever they are
    z2 = z.clone()
    z2[~m] = float("nan")
    again = pkg.ops.router_balance(z2.to(dev), idx.to(dev), m.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(again, (loss, counts, probs, tokens)))
    g2 = pkg.ops.router_balance_vjp(z2.to(dev), idx.to(dev), counts, tokens,
                                    torch.tensor(1.0, device=dev), m.to(dev), dw.to(dev))
    assert torch.equal(g2, got)


@gpu
@pytest.mark.parametrize("T", [6, 600])
def test_infinite_logits_and_bad_indices(pkg, dev, T):
    """Experts shut off by -inf, the type's lowest value, rows with nothing
    left, indices out of range."""
    z, idx, _ = inputs(T, T, 70, 5)
    z[:, 3] = float("-inf")
    z[1, 5:] = torch.finfo(torch.float32).min
    z[2] = float("-inf")
    idx[4, 2], idx[3, 0] = 70, -5
    loss, counts, probs, tokens = pkg.ops.router_balance(z.to(dev), idx.to(dev))
    assert pkg.ops.workspace_status(loss._mlxr_workspace) == 1
    want, c, p, n = forward64(z, idx, None)
    assert torch.equal(counts.cpu().long(), c) and int(tokens) == T == n
    assert float(probs[3]) == 0.0
    fin = torch.where(z < -1e30, torch.zeros_like(z), z)
    tol = rel_p(fin, None) + T * 2.0 ** -24
    assert bool(((probs.cpu().double() - p).abs() <= tol * p).all())
    dw = torch.randn((T, 5), generator=torch.Generator().manual_seed(3))
    got = pkg.ops.router_balance_vjp(z.to(dev), idx.to(dev), counts, tokens,
                                     torch.tensor(0.5, device=dev), None, dw.to(dev)).cpu()
    ref, mass = vjp64(z, idx, None, 0.5, dw)
    assert bool(((got.double() - ref).abs() <= (3 * tol + 90 * 2.0 ** -23) * mass + 1e-38).all())
    assert bool((got[2] == 0).all()) and bool(torch.isfinite(got).all())
    idx[4, 2], idx[3, 0] = 0, 0
    loss, *_ = pkg.ops.router_balance(z.to(dev), idx.to(dev))
    assert pkg.ops.workspace_status(loss._mlxr_workspace) == 0


@gpu
def test_empty_strided_and_batched(pkg, dev):
    ops = pkg.ops
    z = torch.zeros((0, 8), device=dev)
    loss, counts, probs, tokens = ops.router_balance(
        z, torch.zeros((0, 2), dtype=torch.int32, device=dev))
    assert float(loss) == 0 and int(tokens) == 0 and int(counts.sum()) == 0
    assert float(probs.sum()) == 0
    assert ops.router_balance_vjp(z, torch.zeros((0, 2), dtype=torch.int32, device=dev), counts,
                                  tokens, loss).shape == (0, 8)
    # logits as columns of a wider tensor (a shared gate beside them), tokens
    # in two axes, int64 indices, a uint8 mask
    z, idx, m = inputs(3, 600, 48, 4, mask="some")
    wide = torch.full((600, 49), float("nan"))
    wide[:, :48] = z
    a = ops.router_balance(z.to(dev), idx.to(dev), m.to(dev))
    b = ops.router_balance(wide.to(dev)[:, :48], idx.to(dev).long(), m.to(dev).to(torch.uint8))
    c = ops.router_balance(z.to(dev).view(3, 200, 48), idx.to(dev).view(3, 200, 4),
                           m.to(dev).view(3, 200))
    d = ops.router_balance(z.t().contiguous().to(dev).t(), idx.to(dev), m.to(dev))
    for other in (b, c, d):
        assert all(torch.equal(x, y) for x, y in zip(a, other))
    one = torch.ones((), device=dev)
    ga = ops.router_balance_vjp(z.to(dev), idx.to(dev), a[1], a[3], one, m.to(dev))
    gb = ops.router_balance_vjp(wide.to(dev)[:, :48], idx.to(dev), a[1], a[3], one, m.to(dev))
    gc = ops.router_balance_vjp(z.to(dev).view(3, 200, 48), idx.to(dev).view(3, 200, 4), a[1],
                                a[3], one, m.to(dev).view(3, 200))
    assert torch.equal(ga, gb) and torch.equal(ga, gc.view(600, 48))


@gpu
def test_gradient_against_differences(pkg, dev):
    """Central differences of the kernel's own forward (counts held by the
    fixed choices), along random directions.  The loss is f32: its rounding
    over the step bounds the difference's error."""
    ops = pkg.ops
    z, idx, m = inputs(11, 40, 16, 4, mask="some")
    loss, counts, _, tokens = ops.router_balance(z.to(dev), idx.to(dev), m.to(dev))
    grad = ops.router_balance_vjp(z.to(dev), idx.to(dev), counts, tokens,
                                  torch.ones((), device=dev), m.to(dev)).cpu().double()
    g = torch.Generator().manual_seed(5)
    for _ in range(4):
        v = torch.randn((40, 16), generator=g)
        h = 2.0 ** -6
        up = ops.router_balance((z + h * v).to(dev), idx.to(dev), m.to(dev))[0]
        dn = ops.router_balance((z - h * v).to(dev), idx.to(dev), m.to(dev))[0]
        diff = (float(up) - float(dn)) / (2 * h)
        want = float((grad * v.double()).sum())
        # third order: each row's softmax along v, |v|_inf^3 at most, averaged
        third = float(v.double().abs().max() ** 3) * float(loss) * h * h
        noise = 4 * (rel_p(z, m) + 40 * 2.0 ** -24) * float(loss) / h
        assert abs(diff - want) <= third + noise


@gpu
@pytest.mark.parametrize("T", [40, 3000])
def test_equal_bits_graph_and_streams(pkg, dev, T):
    ops = pkg.ops
    z, idx, m = (v.to(dev) for v in inputs(2, T, 128, 8, mask="some"))
    dw = torch.randn((T, 8), device=dev)
    one = torch.ones((), device=dev)

    def step():
        loss, counts, probs, tokens = ops.router_balance(z, idx, m)
        dz = ops.router_balance_vjp(z, idx, counts, tokens, one, m, dw)
        return [loss, counts, probs, tokens, dz]

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        z.mul_(1.1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager))


@gpu
@pytest.mark.parametrize("T", [12, 600])
def test_router_step_over_mxfp4_experts(pkg, dev, T):
    """The operators together, as a router is tuned over frozen quantised
    experts: route, mxfp4 experts, weighted sum, a loss on the output plus the
    balance loss; the gradient in the router's weight against torch's in 64
    bits from the same expert outputs."""
    ops, nn = pkg.ops, pkg.nn
    E, d, f, K = 16, 256, 128, 4
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, d), generator=g).bfloat16().to(dev)
    gate = (torch.randn((E, d), generator=g) * 0.1).to(dev)
    ffn = nn.SplitSwitchFfn.from_dense(*[
        (torch.randn(s, generator=g) * 0.05).bfloat16().to(dev)
        for s in ((E, f, d), (E, f, d), (E, d, f))], mode="mxfp4")
    up = torch.randn((T, d), generator=g).to(dev)  # d loss / d output
    keep = (torch.rand(T, generator=g) < 0.8).to(dev)
    up = up * keep[:, None]
    coef = torch.tensor(0.05, device=dev)

    idx, w, logits = ops.router_topk(x, gate, K, return_logits=True)
    assert logits.shape == (T, E)
    y = ffn.forward(x, idx)
    _, counts, _, tokens = ops.router_balance(logits, idx, keep)
    dw = (y.float() * up[:, None, :]).sum(-1)
    dz = ops.router_balance_vjp(logits, idx, counts, tokens, coef, keep, dw)
    dgate = dz.double().t() @ x.double()

    gate64 = gate.double().requires_grad_()
    z = x.double() @ gate64.t()
    assert float((z.detach() - logits.double()).abs().max()) < 1e-4
    p = torch.softmax(z, 1)
    top = p.gather(1, idx.long())
    w64 = top / top.sum(1, keepdim=True)
    assert float((w64.detach() - w.double()).abs().max()) < 1e-4
    out = (w64[:, :, None] * y.double()).sum(1)
    n = keep.sum()
    fe = torch.nn.functional.one_hot(idx.long(), E).sum(1).double()[keep].sum(0) / (n * K)
    aux = E * (fe * (p * keep[:, None]).sum(0) / n).sum()
    ((out * up.double()).sum() + coef.double() * aux).backward()
    # logits and dw are f32 sums of d terms: relative to the gradient's mass
    mass = (dz.double().abs().t() @ x.double().abs())
    assert bool(((dgate - gate64.grad).abs() <= 1e-4 * (mass + mass.mean())).all())


@gpu
@pytest.mark.parametrize("T", [6, 600])
@pytest.mark.parametrize("E", [8, 60, 65, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_a_softmax(pkg, dev, T, E, dtype):
    """NaN and +inf logits in rows that count make the row, the loss and the
    mean probabilities NaN, as the formula does, whether or not the experts
    fill the lanes; the other rows' gradients are as without them, and a row of
    -inf alone still has none."""
    ops, K, inf, nan = pkg.ops, 4, float("inf"), float("nan")
    z, idx, _ = inputs(T + E, T, E, K, dtype)
    bad = z.clone()
    bad[0] = nan                # nothing but NaN
    bad[1] = -inf               # NaN beside experts that are shut off
    bad[1, idx[1, 2].long()] = nan
    bad[2, idx[2, 0].long()] = inf
    bad[3, idx[3, 1].long()] = nan
    bad[4] = -inf
    idx, dw = idx.to(dev), torch.randn((T, K), generator=torch.Generator().manual_seed(E)).to(dev)
    one = torch.ones((), device=dev)
    _, counts, _, tokens = ops.router_balance(z.to(dev), idx)
    for rows in ([0], [1], [2], [3], [0, 1, 2, 3, 4]):
        zr = z.clone()
        zr[rows] = bad[rows]
        loss, c, probs, n = ops.router_balance(zr.to(dev), idx)
        assert bool(torch.isnan(loss)) and bool(torch.isnan(probs).all())
        assert torch.equal(c, counts) and int(n) == T
    bad = bad.to(dev)
    both = ops.router_balance_vjp(bad, idx, counts, tokens, one, None, dw)
    loss_only = ops.router_balance_vjp(bad, idx, counts, tokens, one)
    dw_only = ops.router_balance_vjp(bad, idx, dweights=dw)
    assert bool(torch.isnan(both[:4]).all()) and bool(torch.isnan(loss_only[:4]).all())
    # the weights' term reaches the chosen experts only
    hit = torch.zeros((T, E), dtype=torch.bool, device=dev).scatter(1, idx.long(), True)
    assert torch.equal(torch.isnan(dw_only[:4]), hit[:4])
    for got, kw in ((both, (counts, tokens, one, None, dw)), (loss_only, (counts, tokens, one)),
                    (dw_only, (None, None, None, None, dw))):
        assert bool((got[4] == 0).all())
        assert torch.equal(got[5:], ops.router_balance_vjp(z.to(dev), idx, *kw)[5:])


@gpu
def test_nan_outside_the_chosen_experts(pkg, dev):
    """The weights' term is a softmax of the chosen logits alone: what the other
    experts of the row hold does not reach it."""
    z, idx, _ = inputs(9, 20, 60, 3)
    dw = torch.randn((20, 3), generator=torch.Generator().manual_seed(2)).to(dev)
    bad = z.clone()
    hit = torch.zeros((20, 60), dtype=torch.bool).scatter(1, idx.long(), True)
    bad[~hit] = float("nan")
    idx = idx.to(dev)
    assert torch.equal(pkg.ops.router_balance_vjp(bad.to(dev), idx, dweights=dw),
                       pkg.ops.router_balance_vjp(z.to(dev), idx, dweights=dw))


@gpu
def test_one_token_without_a_row_axis(pkg, dev):
    """Logits [E] with choices [K] are one token; its mask has no axis."""
    ops = pkg.ops
    z, idx, _ = inputs(4, 1, 60, 3)
    z, idx, one = z.to(dev), idx.to(dev), torch.ones((), device=dev)
    dw = torch.randn((1, 3), generator=torch.Generator().manual_seed(6)).to(dev)
    for m in (None, torch.ones(1, dtype=torch.bool, device=dev),
              torch.zeros(1, dtype=torch.bool, device=dev)):
        m0 = None if m is None else m[0]
        want = ops.router_balance(z, idx, m)
        got = ops.router_balance(z[0], idx[0], m0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        dz = ops.router_balance_vjp(z, idx, want[1], want[3], one, m, dw)
        d0 = ops.router_balance_vjp(z[0], idx[0], want[1], want[3], one, m0, dw[0])
        assert d0.shape == (60,) and torch.equal(d0, dz[0])


@gpu
@pytest.mark.parametrize("T", [5, 600])
def test_indices_past_32_bits(pkg, dev, T):
    """64-bit indices that no 32-bit one holds are out of range: not counted,
    without a gradient, and the status word says so."""
    ops = pkg.ops
    z, idx, _ = inputs(T, T, 24, 3)
    wide, cut = idx.long(), idx.clone()
    wide[0, 0], wide[1, 2], wide[2, 1], wide[4, 0] = 2 ** 32 + 5, -2 ** 32, 2 ** 31, 2 ** 63 - 1
    cut[0, 0] = cut[1, 2] = cut[2, 1] = cut[4, 0] = 24
    a, b = ops.router_balance(z.to(dev), wide.to(dev)), ops.router_balance(z.to(dev), cut.to(dev))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert ops.workspace_status(a[0]._mlxr_workspace) == 1
    dw = torch.randn((T, 3), generator=torch.Generator().manual_seed(8)).to(dev)
    assert torch.equal(ops.router_balance_vjp(z.to(dev), wide.to(dev), dweights=dw),
                       ops.router_balance_vjp(z.to(dev), cut.to(dev), dweights=dw))


def test_routers_refuse_other_types_and_widths(pkg):
    """What the kernels would read past its end, or as another type."""
    ops, nn, Err = pkg.ops, pkg.nn, pkg.MlxrMoeError
    x, gate = torch.zeros(4, 64).bfloat16(), torch.zeros(8, 64)
    with pytest.raises(Err, match="gate_w must be float32"):
        ops.router_topk(x, gate.bfloat16(), 2)
    with pytest.raises(Err, match="gate_w must be float32"):
        ops.router_topk(x, gate[0], 2)
    with pytest.raises(Err, match="last dim must be 32"):
        ops.router_topk(x, gate[:, :32], 2)
    with pytest.raises(Err, match="x must be bfloat16"):
        ops.router_topk(x.float(), gate, 2)
    with pytest.raises(Err, match="ROCm device"):
        ops.router_topk(x, gate, 2)
    bf = nn.Linear(gate.bfloat16())
    with pytest.raises(Err, match="last dim must be 64"):
        ops.router_topk_quantized(x[:, :32], bf, 2)
    with pytest.raises(Err, match="x must be bfloat16"):
        ops.router_topk_quantized(x.float(), bf, 2)
    with pytest.raises(Err, match="ROCm device"):
        ops.router_topk_quantized(x, bf, 2)


@gpu
@pytest.mark.parametrize("T,E,d,K", [(1, 8, 128, 2), (33, 60, 512, 4), (1536, 128, 2048, 8)])
@pytest.mark.parametrize("form", ["f32", "q8", "q4", "bf16"])
def test_logits_a_router_returns(pkg, dev, T, E, d, K, form):
    """Every router form's logits are the products its choices were made of:
    bf16 values where the router is one of bf16, the choices their largest, the
    weights the softmax of those."""
    ops, nn = pkg.ops, pkg.nn
    g = torch.Generator().manual_seed(T + E)
    x = torch.randn((T, d), generator=g).bfloat16().to(dev)
    w = (torch.randn((E, d), generator=g) * 0.05).to(dev)
    if form == "f32":
        idx, wts, z = ops.router_topk(x, w, K, return_logits=True)
    else:
        lin = nn.Linear(w.bfloat16())
        w = lin.weight[0]
        if form != "bf16":
            lin = nn.QuantizedLinear.try_from_linear(w, bits=int(form[1]))
            w = ops.dequantize(lin.weight[0], lin.scales[0], lin.biases[0], bits=lin.bits,
                               out_dtype=torch.float32)
        idx, wts, z = ops.router_topk_quantized(x, lin, K, return_logits=True)
        assert torch.equal(z.bfloat16().float(), z)
    assert z.shape == (T, E) and z.dtype == torch.float32
    want, mass = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    # an f32 sum of d products and one rounding to bf16; quantised, codes times scale and
    # biases may be summed apart, their magnitudes |w| + 2 |bias| at most
    if form[0] == "q":
        bias = lin.biases[0].double().abs().repeat_interleave(64, 1)
        mass = mass + 2 * x.double().abs() @ bias.t()
    tol = (d + 4) * 2.0 ** -23 * mass
    if form != "f32":
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((z.double() - want).abs() <= tol).all())
    # the choices: no other expert's probability is larger, but by two roundings of them
    # to bf16 where the router works in that
    p = torch.softmax(z.double(), 1)
    top = p.gather(1, idx.long())
    half = 0.0 if form == "f32" else 2.0 ** -8
    room = (1.0 + half) / (1.0 - half) * (1.0 + 2 * rel_p(z.cpu(), None))
    rest = p.scatter(1, idx.long(), 0.0).amax(1)
    assert bool((rest <= top.amin(1) * room).all())
    # the weights from these logits: each probability, their sum and the quotient rounded
    rel = 2 * rel_p(z.cpu(), None) + (K + 3) * (2.0 ** -24 if form == "f32" else 2.0 ** -8)
    want = top / top.sum(1, keepdim=True)
    assert bool(((wts.double() - want).abs() <= rel * want).all())
    # and on to the balance loss
    check_forward(ops, dev, z.cpu(), idx.cpu(), None)
