"""add_rms_norm (the residual add with RMSNorm, its output in bf16 or in mode mxfp8),
its gradients, and quantize / dequantize in mode mxfp8, against plain 64-bit
restatements of their formulas.

Tolerances: a sum of d terms in f32 is off by at most d * 2^-24 of the sum of the
terms' magnitudes, and the quotient, the root, its inverse and the products add a few
roundings of 2^-24 each (16 are counted).  Storing rounds by 2^-8 (bf16) or 2^-24.
"""
import pytest
import torch

gpu = pytest.mark.gpu
EPS = 1e-6
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rel(d):
    return (d + 16) * 2.0 ** -24


def inputs(seed, T, d, xt=torch.bfloat16, ht=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, d), generator=g).to(xt)
    res = (torch.randn((T, d), generator=g) * torch.exp(torch.randn(d, generator=g))).to(ht)
    w = (1 + 0.3 * torch.randn(d, generator=g)).bfloat16()
    return x, res, w


def norm64(h, w, eps=EPS):
    h = h.double()
    return w.double() * h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)


# ------------------------------------------------------------- mode mxfp8, by hand
def scale_bytes8(v):
    """Scale byte of each group of 32 of v (f64 [.., cols], finite)."""
    top = v.unflatten(-1, (-1, 32)).abs().amax(-1)
    return (torch.frexp(top).exponent - 1 - 8 + 127).clamp_min(0).where(top > 0, torch.tensor(0))


def nearest8(v, byte):
    """v [.., cols] f64 rounded to e4m3 values under the given scale bytes."""
    s = torch.ldexp(torch.ones_like(v), byte.repeat_interleave(32, -1) - 127)
    a = v.abs() / s
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp_max(448.0), v) * s


def decode8(words, byte):
    """e4m3 words and scale bytes as f64 values, from the format's definition."""
    b = torch.stack([(words.long() >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2)
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double()))
    v = torch.where((b & 127) == 127, torch.nan, v)
    v = torch.where(b > 127, -v, v)
    s = torch.ldexp(torch.ones_like(v), byte.long().repeat_interleave(32, -1) - 127)
    return v * torch.where(byte.repeat_interleave(32, -1) == 255, torch.nan, s)


def values8(kind, shape, dtype):
    g = torch.Generator().manual_seed(len(kind))
    v = torch.randn(shape, generator=g)
    if kind == "wide":  # groups from tiny to huge
        v = v * torch.exp2(torch.randint(-120, 120, shape[:-1] + (1,), generator=g).float())
    if kind == "ties":  # the midpoints between codes, and past the largest code
        v = torch.randint(-1024, 1025, shape, generator=g).float()
    if kind == "small":  # codes below the smallest normal one, subnormal values
        v = v * torch.exp2(torch.randint(-18, 1, shape, generator=g).float())
        v[0] *= 2.0 ** -125
    v[..., -1, :32] = 0.0
    return v.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "wide", "ties", "small"])
@pytest.mark.parametrize("shift", [0, 1])
def test_quantize_mxfp8(pkg, dev, kind, dtype, shift):
    v = values8(kind, (3, 7, 96), dtype)
    flat = torch.zeros(v.numel() + shift, dtype=dtype, device=dev)
    flat[shift:] = v.flatten().to(dev)  # off 16-byte alignment too
    q, sc, none = pkg.ops.quantize(flat[shift:].view(v.shape), mode="mxfp8")
    assert none is None and q.shape == (3, 7, 24) and sc.shape == (3, 7, 3)
    assert q.dtype == torch.int32 and sc.dtype == torch.uint8
    want_sc = scale_bytes8(v.double())
    assert torch.equal(sc.cpu().long(), want_sc.long())
    want = nearest8(v.double(), want_sc)
    assert torch.equal(decode8(q.cpu(), sc.cpu()), want)
    out = pkg.ops.dequantize(q, sc, mode="mxfp8", out_dtype=torch.float32)
    assert torch.equal(out.cpu().double(), want.float().double())
    out = pkg.ops.dequantize(q, sc, mode="mxfp8")
    assert out.dtype == torch.bfloat16 and torch.equal(out.cpu(), want.float().bfloat16())


@gpu
def test_mxfp8_nan_inf_and_every_code(pkg, dev):
    v = torch.ones((4, 64))
    v[0, 3], v[1, 40], v[2, 0] = torch.nan, torch.inf, -torch.inf
    q, sc, _ = pkg.ops.quantize(v.to(dev), mode="mxfp8")
    assert sc.tolist() == [[255, 119], [119, 255], [255, 119], [119, 119]]
    out = pkg.ops.dequantize(q, sc, mode="mxfp8").cpu().view(4, 2, 32)
    bad = torch.tensor([[1, 0], [0, 1], [1, 0], [0, 0]]).bool()
    assert bool(torch.isnan(out[bad]).all()) and bool((out[~bad] == 1).all())
    words = torch.arange(256, dtype=torch.uint8).view(torch.int32).view(1, 64)
    for byte in (0, 1, 100, 127, 200, 254, 255):
        b = torch.full((1, 8), byte, dtype=torch.uint8)
        got = pkg.ops.dequantize(words.to(dev), b.to(dev), mode="mxfp8",
                                 out_dtype=torch.float32).cpu()
        want = decode8(words, b).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5)), byte


# ------------------------------------------------------------------------- forward
SHAPES = [(1, 2048), (1, 8), (3, 1), (5, 37), (7, 520), (4, 4096), (2, 4104), (2, 16384),
          (1, 20000), (2500, 96), (2050, 2048), (2049, 8), (2048, 4096), (2051, 264)]


@gpu
@pytest.mark.parametrize("T,d", SHAPES)
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
def test_add_rms_norm(pkg, dev, T, d, xt, ht):
    x, res, w = inputs(T + d, T, d, xt, ht)
    h, y = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev), EPS)
    assert h.dtype == ht and y.dtype == torch.bfloat16
    assert torch.equal(h.cpu(), (x.float() + res.float()).to(ht))
    want = norm64(h.cpu(), w)
    tol = (rel(d) + 2.0 ** -8) * want.abs() + 1e-38
    assert bool(((y.cpu().double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("T,d", [(1, 2048), (3, 32), (5, 96), (2, 4128), (1, 20000), (2300, 64),
                                 (2048, 2048)])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
def test_add_rms_norm_mxfp8(pkg, dev, T, d, xt, ht):
    x, res, w = inputs(T + d, T, d, xt, ht)
    w[: d // 32 * 16] = 0  # groups of zeros
    h, q, sc = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev), EPS, mode="mxfp8")
    assert q.shape == (T, d // 4) and sc.shape == (T, d // 32)
    assert torch.equal(h.cpu(), (x.float() + res.float()).to(ht))
    y = norm64(h.cpu(), w)
    lo, hi = y * (1 - rel(d)), y * (1 + rel(d))
    byte, blo, bhi = sc.cpu().long(), scale_bytes8(lo), scale_bytes8(hi)
    assert bool(((byte == blo) | (byte == bhi)).all())
    a, b = nearest8(lo, byte), nearest8(hi, byte)
    got = decode8(q.cpu(), sc.cpu())
    assert bool(((torch.minimum(a, b) <= got) & (got <= torch.maximum(a, b))).all())


@gpu
def test_add_rms_norm_views_and_shapes(pkg, dev):
    x, res, w = inputs(1, 6, 256)
    wide = torch.zeros((6, 300), dtype=torch.bfloat16, device=dev)
    wide[:, 3:259] = x.to(dev)
    one = torch.zeros(256 + 1, dtype=torch.bfloat16, device=dev)
    one[1:] = w.to(dev)  # a weight off 16-byte alignment
    h0, y0 = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev))
    h1, y1 = pkg.ops.add_rms_norm(wide[:, 3:259].view(2, 3, 256), res.to(dev).view(2, 3, 256),
                                  one[1:])
    assert h1.shape == y1.shape == (2, 3, 256)
    assert torch.equal(h0, h1.view(6, 256))
    want = norm64(h0.cpu(), w)
    assert bool(((y1.view(6, 256).cpu().double() - want).abs()
                 <= (rel(256) + 2.0 ** -8) * want.abs()).all())
    h2, y2 = pkg.ops.add_rms_norm(x[0].to(dev), res[0].to(dev), w.to(dev))
    assert h2.shape == (256,) and torch.equal(y2, y0[0])
    for mode in (None, "mxfp8"):
        got = pkg.ops.add_rms_norm(x[:0].to(dev), res[:0].to(dev), w.to(dev), mode=mode)
        assert got[0].shape == (0, 256) and got[1].shape[0] == 0


@gpu
def test_add_rms_norm_special_values(pkg, dev):
    x, res, w = inputs(2, 6, 64)
    x[1, 5], res[2, 7], x[3, 9] = torch.nan, torch.inf, -torch.inf
    x[4], res[4] = 0, 0
    h, y = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev), 0.0)
    y = y.cpu()
    assert bool(torch.isnan(y[1]).all())
    for t, j in ((2, 7), (3, 9)):  # r is 0: the infinity gives NaN, the others 0
        assert bool(torch.isnan(y[t, j])) and int(torch.isnan(y[t]).sum()) == 1
        assert int((y[t] == 0).sum()) == 63
    assert bool(torch.isnan(y[4]).all())  # 0 / 0 without eps
    h, y = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev), EPS)
    assert bool((y[4] == 0).all())
    _, q, sc = pkg.ops.add_rms_norm(x.to(dev), res.to(dev), w.to(dev), EPS, mode="mxfp8")
    assert sc[1].tolist() == [255, 255] and sc[2].tolist() == [255, 0]
    assert sc[4].tolist() == [0, 0] and bool((q[4] == 0).all())


# ------------------------------------------------------------------------ gradients
def vjp64(dy, h, w, dh, eps=EPS):
    dy, h, w = dy.double(), h.double(), w.double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = dy * w
    c = (g * h).mean(-1, keepdim=True)
    dx = r * (g - h * r * r * c)
    mass = r * (g.abs() + h.abs() * r * r * (g * h).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, mass = dx + dh.double(), mass + dh.double().abs()
    return dx, mass, (dy * h * r).sum(0), (dy * h * r).abs().sum(0)


@gpu
@pytest.mark.parametrize("T,d", SHAPES + [(5000, 2048), (70, 33), (130, 300)])
@pytest.mark.parametrize("yt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_dh", [True, False])
def test_add_rms_norm_vjp(pkg, dev, T, d, yt, ht, with_dh):
    dy, h, w = inputs(T * 3 + d, T, d, yt, ht)
    dh = inputs(T + 7 * d, T, d, ht)[0] if with_dh else None
    dx, dw = pkg.ops.add_rms_norm_vjp(dy.to(dev), h.to(dev), w.to(dev), EPS,
                                      None if dh is None else dh.to(dev))
    assert dx.dtype == ht and dw.dtype == torch.float32 and dw.shape == (d,)
    want, mass, want_w, mass_w = vjp64(dy, h, w, dh)
    # r enters cubed, and c is a sum of its own
    tol = 4 * rel(d) * mass
    tol = tol + HALF[ht] * (want.abs() + tol) + 1e-38
    assert bool(((dx.cpu().double() - want).abs() <= tol).all())
    tol = (rel(d) + rel(T)) * mass_w + 1e-38
    assert bool(((dw.cpu().double() - want_w).abs() <= tol).all())


@gpu
def test_add_rms_norm_vjp_against_differences(pkg, dev):
    """<dx, v> and <dweight, u> against central differences of the plain forward pass."""
    T, d = 5, 40
    dy, h, w = inputs(11, T, d, torch.float32, torch.float32)
    dx, dw = pkg.ops.add_rms_norm_vjp(dy.to(dev), h.to(dev), w.to(dev), EPS)
    g = torch.Generator().manual_seed(5)
    v = torch.randn((T, d), generator=g, dtype=torch.float64)
    u = torch.randn(d, generator=g, dtype=torch.float64)

    def f(step, wstep):
        hh, ww = h.double() + step * v, w.double() + wstep * u
        return (dy.double() * ww * hh
                / torch.sqrt((hh * hh).mean(-1, keepdim=True) + EPS)).sum()

    e = 1e-4  # the third derivatives are of order 1: an error of order e^2
    for got, dirn, diff in ((dx, v, f(e, 0) - f(-e, 0)), (dw, u, f(0, e) - f(0, -e))):
        got = got.cpu().double()
        mass = float((got * dirn).abs().sum())
        assert abs(float((got * dirn).sum()) - float(diff) / (2 * e)) <= 1e-5 * mass


@gpu
def test_add_rms_norm_vjp_edges(pkg, dev):
    dy, h, w = inputs(3, 4, 64)
    z = pkg.ops.add_rms_norm_vjp(dy[:0].to(dev), h[:0].to(dev), w.to(dev))
    assert z[0].shape == (0, 64) and bool((z[1] == 0).all())
    a = pkg.ops.add_rms_norm_vjp(dy.to(dev), h.to(dev), w.to(dev))
    b = pkg.ops.add_rms_norm_vjp(dy.to(dev).view(2, 2, 64), h.to(dev).view(2, 2, 64), w.to(dev))
    assert b[0].shape == (2, 2, 64)
    assert torch.equal(a[0], b[0].view(4, 64)) and torch.equal(a[1], b[1])


@gpu
def test_add_rms_norm_on_a_stream_and_in_a_graph(pkg, dev):
    ops = pkg.ops
    x, res, w = [t.to(dev) for t in inputs(4, 3000, 512)]
    dy = inputs(5, 3000, 512)[0].to(dev)

    def step():
        h, y = ops.add_rms_norm(x, res, w)
        _, q, sc = ops.add_rms_norm(x, res, w, mode="mxfp8")
        dx, dw = ops.add_rms_norm_vjp(dy, h, w, dh=res)
        return h, y, q, sc, dx, dw

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.copy_(inputs(20 + k, 3000, 512)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------- refusals
def test_refusals(pkg):
    lib, C = pkg._capi.lib(), pkg._capi
    err = pkg._capi.last_error

    def fwd(T=2, d=64, eps=1e-6, mode=None, xd=C.BFLOAT16, rd=C.BFLOAT16, x=16, res=16, w=16,
            h=16, out=16, sc=None):
        return lib.mlxr_moe_add_rms_norm(x, xd, res, rd, T, d, w, eps, mode, h, out, sc, None)

    for kw, word in [(dict(T=-1), "bad shape"), (dict(d=0), "bad shape"),
                     (dict(T=1 << 24), "at most"), (dict(d=(1 << 20) + 1), "at most"),
                     (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                     (dict(mode=b"mxfp4"), "mode"), (dict(xd=2), "f32 or bf16"),
                     (dict(rd=5), "f32 or bf16"), (dict(mode=b"mxfp8", d=48, sc=16), "groups of 32"),
                     (dict(sc=16), "scales go with"), (dict(mode=b"mxfp8"), "null"),
                     (dict(x=None), "null"), (dict(res=None), "null"), (dict(w=None), "null"),
                     (dict(h=None), "null"), (dict(out=None), "null"), (dict(x=17), "aligned"),
                     (dict(rd=C.FLOAT32, h=18), "aligned"), (dict(w=17), "aligned")]:
        assert fwd(**kw) == -1 and word in err(), kw
    assert fwd(T=0) == 0

    def vjp(T=2, d=64, eps=1e-6, yd=C.BFLOAT16, hd=C.BFLOAT16, dy=16, h=16, w=16, dh=None, dx=16,
            dw=16, ws=256, n=1 << 20):
        return lib.mlxr_moe_add_rms_norm_vjp(dy, yd, h, hd, T, d, w, eps, dh, dx, dw, ws, n, None)

    for kw, word in [(dict(T=-1), "bad shape"), (dict(d=0), "bad shape"),
                     (dict(T=1 << 24), "at most"), (dict(eps=-1.0), "eps"),
                     (dict(yd=2), "f32 or bf16"), (dict(hd=2), "f32 or bf16"),
                     (dict(dy=None), "null"), (dict(h=None), "null"), (dict(dx=None), "null"),
                     (dict(dw=None), "null"), (dict(dh=17), "aligned"), (dict(dw=18), "aligned"),
                     (dict(ws=None), "workspace is NULL"), (dict(ws=16), "256-byte"),
                     (dict(n=16), "too small")]:
        assert vjp(**kw) == -1 and word in err(), kw
    assert lib.mlxr_moe_add_rms_norm_vjp_workspace_size(-1, 64) == 0
    OI = C.OptionalInt
    for gs, bits, word in [(64, None, "group_size 32"), (None, 4, "bits 8")]:
        assert lib.mlxr_moe_quantize(16, C.BFLOAT16, 4, 64, OI.of(gs), OI.of(bits), b"mxfp8", 16,
                                     16, None, None) == -1 and word in err()
        assert lib.mlxr_moe_dequantize(16, 16, None, C.UINT8, 4, 64, OI.of(gs), OI.of(bits),
                                       b"mxfp8", 16, C.BFLOAT16, None) == -1 and word in err()
    n = OI.of(None)
    assert lib.mlxr_moe_quantize(16, C.BFLOAT16, 4, 64, n, n, b"mxfp8", 16, 16, 16, None) == -1
    assert "no biases" in err()
    assert lib.mlxr_moe_quantize(16, C.BFLOAT16, 4, 40, n, n, b"mxfp8", 16, 16, None, None) == -1
    assert "multiple" in err()


def test_python_refusals(pkg):
    ops, E = pkg.ops, pkg.MlxrMoeError
    x, w = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(E, match="ROCm device"):
        ops.add_rms_norm(x, x, w)
    with pytest.raises(E, match="ROCm device"):
        ops.add_rms_norm_vjp(x, x, w)
    with pytest.raises(E, match="unsupported mode"):
        ops.add_rms_norm(x, x, w, mode="mxfp4")
    with pytest.raises(E, match="ROCm device"):
        ops.quantize(x, mode="mxfp8")


@gpu
def test_python_refusals_on_the_device(pkg, dev):
    ops, E = pkg.ops, pkg.MlxrMoeError
    x = torch.zeros((2, 48), dtype=torch.bfloat16, device=dev)
    w = torch.zeros(48, dtype=torch.bfloat16, device=dev)
    with pytest.raises(E, match="groups of 32"):
        ops.add_rms_norm(x, x, w, mode="mxfp8")
    with pytest.raises(E, match="must be the same"):
        ops.add_rms_norm(x, x[:1], w)
    with pytest.raises(E, match="weight must be"):
        ops.add_rms_norm(x, x, w.float())
    with pytest.raises(E, match="weight must be"):
        ops.add_rms_norm(x, x, w[:47])
    with pytest.raises(E, match="unsupported dtype"):
        ops.add_rms_norm(x.half(), x, w)
    with pytest.raises(E, match="dh must be"):
        ops.add_rms_norm_vjp(x, x, w, dh=x.float())
    with pytest.raises(E, match="must be the same"):
        ops.add_rms_norm_vjp(x[:1], x, w)
    with pytest.raises(E, match="eps"):
        ops.add_rms_norm(x, x, w, -1.0)
    q, sc, _ = ops.quantize(torch.zeros((2, 64), device=dev), mode="mxfp8")
    with pytest.raises(E, match="eight words"):
        ops.dequantize(q, sc[:, :1], mode="mxfp8")


# The codes go by the value in 64 bits: f32 would put one value in 2^18 on the wrong side of
# the middle of two codes, dozens of these.
@gpu
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d,shift", [(4096, 2048, 0), (600, 8192, 0), (512, 2048, 1)])
def test_codes_are_the_nearest(pkg, dev, T, d, shift, ht):
    x, res, w = (t.to(dev) for t in inputs(77, T, d, torch.float32, ht))
    if shift:  # a weight off 16 bytes: the kernel for single values
        w = torch.cat([w[:shift], w])[shift:]
        assert w.data_ptr() % 16
    h, q, sc = pkg.ops.add_rms_norm(x, res, w, EPS, mode="mxfp8")
    y = norm64(h.cpu(), w.cpu())
    byte = scale_bytes8(y)
    assert torch.equal(sc.cpu().long(), byte.long())
    assert torch.equal(decode8(q.cpu(), sc.cpu()), nearest8(y, byte))


# Rows of any length and at any address take 16-byte accesses with a shorter last piece; rows of
# more than 16384 values single ones.
@gpu
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d,shift", [(3, 16385, 0), (2050, 2047, 1), (2050, 4095, 0), (5, 12345, 3),
                                       (2100, 9, 1), (2048, 264, 1), (7, 520, 1), (3, 16384, 1)])
def test_any_length_and_address(pkg, dev, T, d, shift, ht):
    ops = pkg.ops

    def off(t):  # the same values, `shift` elements off 16 bytes
        flat = torch.zeros(t.numel() + shift, dtype=t.dtype, device=dev)
        flat[shift:] = t.flatten().to(dev)
        return flat[shift:].view(t.shape)

    x, res, w = inputs(d + T, T, d, torch.float32, ht)
    h, y = ops.add_rms_norm(off(x), off(res), off(w), EPS)
    h64 = (x + res.float()).to(ht)
    assert torch.equal(h.cpu(), h64)
    want = norm64(h64, w)
    assert bool(((y.cpu().double() - want).abs() <= (2.0 ** -8 + rel(d)) * want.abs()).all())
    g = torch.Generator().manual_seed(d)
    dy, dh = torch.randn((T, d), generator=g), torch.randn((T, d), generator=g).to(ht)
    dx, dw = ops.add_rms_norm_vjp(off(dy), off(h64), off(w), EPS, off(dh))
    hh, dd, w64 = h64.double(), dy.double(), w.double()
    r = 1 / torch.sqrt((hh * hh).mean(-1, keepdim=True) + EPS)
    gw = dd * w64
    c = (gw * hh).mean(-1, keepdim=True)
    want = r * (gw - hh * r * r * c) + dh.double()
    mass = (r * (gw.abs() + hh.abs() * r * r * (gw * hh).abs().mean(-1, keepdim=True))
            + dh.double().abs())
    assert bool(((dx.cpu().double() - want).abs()
                 <= HALF[ht] * want.abs() + (1 + HALF[ht]) * rel(d) * mass).all())
    want, mass = (dd * hh * r).sum(0), (dd * hh * r).abs().sum(0)
    assert bool(((dw.cpu().double() - want).abs() <= (rel(d) + rel(T)) * mass + 1e-30).all())


# Rows that no registers hold go by a kernel of their own, whose norm is in 64 bits, too.
@gpu
@pytest.mark.parametrize("ht", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d", [(160, 16416), (60, 20000), (3, 65536)])
def test_codes_of_wide_rows_are_the_nearest(pkg, dev, T, d, ht):
    x, res, w = (t.to(dev) for t in inputs(78, T, d, torch.float32, ht))
    h, q, sc = pkg.ops.add_rms_norm(x, res, w, EPS, mode="mxfp8")
    y = norm64(h.cpu(), w.cpu())
    byte = scale_bytes8(y)
    assert torch.equal(sc.cpu().long(), byte.long())
    assert torch.equal(decode8(q.cpu(), sc.cpu()), nearest8(y, byte))


@gpu
@pytest.mark.parametrize("d", [64, 16416])
def test_norms_past_the_range_of_f32_are_infinities(pkg, dev, d):
    h = torch.zeros((2, d), dtype=torch.bfloat16)
    h[0, 3], h[1, 40] = float(d) ** 0.5, 1.0
    w = torch.ones(d, dtype=torch.bfloat16)
    w[3], w[40] = 3e38, -1e30
    _, q, sc = pkg.ops.add_rms_norm(torch.zeros_like(h).to(dev), h.to(dev), w.to(dev), 0.0, "mxfp8")
    assert sc[0, 0] == 255 and bool((q[0, :8] == 0).all()) and bool((sc[0, 1:] == 0).all())
    y = norm64(h, w, 0.0)[1:]
    assert torch.equal(sc[1:].cpu().long(), scale_bytes8(y).long())
    assert torch.equal(decode8(q[1:].cpu(), sc[1:].cpu()), nearest8(y, scale_bytes8(y)))
