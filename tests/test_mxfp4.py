"""Mode "mxfp4" (microscaled 4-bit weights): quantise, dequantise, gather_qmm
and the expert modules, against plain 64-bit restatements of their formulas.

Tolerances: a bf16 result is off by half a step of its value at most, 2^-8 of
it; a sum of K products in f32 by K * 2^-23 of the sum of their magnitudes at
most (each of K additions by a step of what has been added so far).  Quantised
and dequantised values are exact.
"""
import ctypes

import pytest
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
gpu = pytest.mark.gpu


# ------------------------------------------------------------ 64-bit formulas
def values64(wq, sc):
    """The weights of packed words [.., K/8] and scale bytes [.., K/32]."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64)
    words = wq.cpu().long() & 0xFFFFFFFF
    code = torch.stack([(words >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2)
    b = sc.cpu().long()
    scale = ((b + 896) << 52).view(torch.float64)  # 2^(b - 127)
    scale = torch.where(b == 255, torch.full_like(scale, float("nan")), scale)
    return table[code] * scale.repeat_interleave(32, -1)


def quantise64(w):
    """(values, scale bytes) of the nearest representable weights, by search
    over the eight magnitudes."""
    v = w.cpu().double().unflatten(-1, (-1, 32))
    big = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    ok = torch.where(bad, torch.ones_like(big), big)
    # floor(log2 big) from the f64's exponent field (big is a normal f64 or 0)
    ex = ((ok.view(torch.int64) >> 52) & 0x7FF) - 1023
    byte = (ex - 2 + 127).clamp_min(0)
    unit = ((byte + 896) << 52).view(torch.float64)
    a = v.abs() / unit[..., None]
    mags = torch.tensor(E2M1, dtype=torch.float64)
    d = (a[..., None] - mags).abs()
    best = d.amin(-1, keepdim=True)
    # ties: the even code
    odd = torch.arange(8) % 2
    code = torch.where(d == best, odd, 2).argmin(-1)
    out = torch.copysign(mags[code], v) * unit[..., None]
    out = torch.where(bad[..., None], torch.full_like(out, float("nan")), out)
    return out.flatten(-2), torch.where(bad, torch.full_like(byte, 255), byte)


def bank(g, shape, std=0.02):
    """Random codes and scales around std: [E, N, K/8] int32, [E, N, K/32]."""
    E, N, K = shape
    wq = torch.randint(-2 ** 31, 2 ** 31 - 1, (E, N, K // 8), generator=g, dtype=torch.int64)
    base = 127 + int(torch.tensor(std / 3.0).log2().floor())
    sc = torch.randint(base - 2, base + 3, (E, N, K // 32), generator=g)
    return wq.to(torch.int32), sc.to(torch.uint8)


def check_sum(y, x64, w64, K):
    """y [.., N] against x64 [.., K] @ w64 [N, K]^T, one bf16 rounding of an
    f32 sum."""
    want = x64 @ w64.t()
    mass = x64.abs() @ w64.abs().t()
    err = (y.double() - want).abs()
    slack = K * 2.0 ** -23 * mass
    bound = 2.0 ** -8 * (want.abs() + slack) + slack
    worst = float((err - bound).max()) if err.numel() else -1.0
    assert worst <= 0, f"error {float(err.max()):.3e} past its bound by {worst:.3e}"


# ------------------------------------------------------------------ refusals
def test_quantize_and_dequantize_refuse(pkg):
    lib, C = pkg._capi.lib(), pkg._capi
    OI = C.OptionalInt

    def q(gs=None, bits=None, cols=64, dt=C.BFLOAT16, biases=None, w=16, wq=16):
        return lib.mlxr_moe_quantize(w, dt, 4, cols, OI.of(gs), OI.of(bits), b"mxfp4", wq, 16,
                                     biases, None)

    assert q(gs=64) == -1 and "group_size 32" in C.last_error()
    assert q(bits=8) == -1 and "bits 4" in C.last_error()
    assert q(cols=48) == -1 and "multiple of group_size 32" in C.last_error()
    assert q(dt=C.UINT8) == -1 and "dtype" in C.last_error()
    assert q(biases=16) == -1 and "no biases" in C.last_error()
    assert q(w=None) == -1 and "null array" in C.last_error()
    assert q(w=17) == -1 and "aligned" in C.last_error()
    assert q(wq=18) == -1 and "aligned" in C.last_error()

    def dq(dt=C.UINT8, biases=None, cols=64, out=16, odt=C.FLOAT32, bits=None):
        return lib.mlxr_moe_dequantize(16, 16, biases, dt, 4, cols, OI.of(32), OI.of(bits),
                                       b"mxfp4", out, odt, None)

    assert dq(dt=C.BFLOAT16) == -1 and "uint8 scales" in C.last_error()
    assert dq(biases=16) == -1 and "no biases" in C.last_error()
    assert dq(cols=40) == -1 and "bad shape" in C.last_error()
    assert dq(bits=8) == -1 and "bits 4" in C.last_error()
    assert dq(out=None) == -1 and "null array" in C.last_error()
    assert dq(out=18) == -1 and "aligned" in C.last_error()
    assert dq(odt=C.UINT8) == -1 and "out" in C.last_error()
    # an empty array needs no memory
    assert lib.mlxr_moe_quantize(None, C.BFLOAT16, 0, 64, OI.of(None), OI.of(None), b"mxfp4",
                                 None, None, None, None) == 0
    assert lib.mlxr_moe_quantize(16, C.BFLOAT16, 4, 64, OI.of(None), OI.of(None), b"nvfp4", 16,
                                 16, None, None) == -1
    assert "mode" in C.last_error()


def test_gather_qmm_refuses(pkg):
    lib, C = pkg._capi.lib(), pkg._capi
    OI = C.OptionalInt

    def call(K=128, N=64, sdt=C.UINT8, biases=None, scales=16, x=16, w=16, gs=None, bits=None,
             transpose=1, rhs=16, E=4):
        return lib.mlxr_moe_gather_qmm(x, C.BFLOAT16, 1, 1, K, w, scales, biases, sdt, E, N,
                                       None, rhs, 1, transpose, OI.of(gs), OI.of(bits), b"mxfp4",
                                       0, 16, C.BFLOAT16, None, 0, None)

    assert call(sdt=C.BFLOAT16) == -1 and "uint8 scales" in C.last_error()
    assert call(biases=16) == -1 and "no biases" in C.last_error()
    assert call(scales=None) == -1 and "null array" in C.last_error()
    assert call(gs=64) == -1 and "group_size 32" in C.last_error()
    assert call(bits=8) == -1 and "bits 4" in C.last_error()
    assert call(transpose=0) == -1 and "transpose" in C.last_error()
    assert call(K=96) == -1 and "multiples of 64" in C.last_error()
    assert call(N=96) == -1 and "multiples of 64" in C.last_error()
    assert call(K=4160) == -1 and "K above" in C.last_error()
    assert call(E=1025) == -1 and "num_experts" in C.last_error()
    assert call(x=8) == -1 and "aligned" in C.last_error()
    assert call(w=None) == -1 and "null array" in C.last_error()
    assert call(scales=18) == -1 and "4-byte aligned" in C.last_error()
    assert call() == -1 and "workspace" in C.last_error()


def test_descriptors_refuse(pkg):
    C = pkg._capi
    lib = C.lib()
    M = C.BITS_MXFP4
    gate = C.QLinear(16, 16, None, 8, 256, 512, 32, M)
    down = C.QLinear(16, 16, None, 8, 512, 256, 32, M)

    def glu(g, u, d):
        ffn = C.SwitchGlu(g, u, d)
        return lib.mlxr_moe_switch_glu_forward(ctypes.byref(ffn), None, 1, None, None, 2, None,
                                               None, 0, None)

    assert glu(gate, gate, down) == -1 and "null array" in C.last_error()
    assert glu(C.QLinear(16, 16, 16, 8, 256, 512, 32, M), gate, down) == -1
    assert "no biases" in C.last_error()
    assert glu(C.QLinear(16, None, None, 8, 256, 512, 32, M), gate, down) == -1
    assert "weight and scales" in C.last_error()
    assert glu(C.QLinear(16, 18, None, 8, 256, 512, 32, M), gate, down) == -1
    assert "4-byte aligned" in C.last_error()
    assert glu(C.QLinear(16, 16, None, 8, 256, 512, 64, M), gate, down) == -1
    assert "group_size must be 32" in C.last_error()
    assert glu(gate, gate, C.QLinear(16, 16, 16, 8, 512, 256, 64, 4)) == -1
    assert "share bits" in C.last_error()
    # routers and gates stay affine, dense or f32
    g = C.QLinear(16, 16, None, 1, 128, 2048, 32, M)
    assert lib.mlxr_moe_router_topk_quantized(None, 1, ctypes.byref(g), 8, None, None, None, 0,
                                              None) == -1
    assert "bits must be 4 or 8" in C.last_error()


def test_python_refuses(pkg):
    ops, nn, Err = pkg.ops, pkg.nn, pkg.MlxrMoeError
    wq = torch.zeros((4, 64, 16), dtype=torch.int32)
    sc = torch.zeros((4, 64, 4), dtype=torch.uint8)
    with pytest.raises(Err, match="mode"):
        ops.quantize(torch.zeros(2, 64), mode="nvfp4")
    with pytest.raises(Err, match="ROCm device"):
        ops.quantize(torch.zeros(2, 64), mode="mxfp4")
    with pytest.raises(Err, match="no biases"):
        nn.QuantizedSwitchLinear(wq, sc, sc, mode="mxfp4")
    with pytest.raises(Err, match="uint8"):
        nn.QuantizedSwitchLinear(wq, sc.bfloat16(), mode="mxfp4")
    with pytest.raises(Err, match="one byte"):
        nn.QuantizedSwitchLinear(wq, sc[:, :, :3], mode="mxfp4")
    with pytest.raises(Err, match="one byte"):
        nn.QuantizedSwitchLinear(wq, sc[:2], mode="mxfp4")
    with pytest.raises(Err, match="group_size 32"):
        nn.QuantizedSwitchLinear(wq, sc, None, 64, 4, "mxfp4")
    with pytest.raises(Err, match="biases are required"):
        nn.QuantizedSwitchLinear(wq, sc.bfloat16())
    m = nn.QuantizedSwitchLinear(wq, sc, mode="mxfp4")
    d = m.descriptor()
    assert (d.bits, d.group_size, d.biases, d.input_dims) == (0x104, 32, None, 128)


# -------------------------------------------------------------------- loader
def write_checkpoint(path, E=8, d=256, f=128, mode="mxfp4"):
    """One layer with mxfp4 experts and shared expert, an affine 8-bit router
    and shared gate named by overrides."""
    import json
    st = pytest.importorskip("safetensors.torch")
    g = torch.Generator().manual_seed(3)
    pre = "language_model.model.layers.2.mlp."
    t = {}
    for name, shape in (("switch_mlp.gate_proj", (E, f, d)), ("switch_mlp.up_proj", (E, f, d)),
                        ("switch_mlp.down_proj", (E, d, f)), ("shared_expert.gate_proj", (f, d)),
                        ("shared_expert.up_proj", (f, d)), ("shared_expert.down_proj", (d, f))):
        wq, sc = bank(g, (1,) * (3 - len(shape)) + shape)
        t[pre + name + ".weight"] = wq.reshape(shape[:-1] + (-1,)).view(torch.uint32)
        t[pre + name + ".scales"] = sc.reshape(shape[:-1] + (-1,))
    q = {"group_size": 32, "bits": 4, "mode": mode}
    for name, rows in (("gate", E), ("shared_expert_gate", 1)):
        t[pre + name + ".weight"] = torch.randint(0, 2 ** 31 - 1, (rows, d // 4), generator=g,
                                                  dtype=torch.int32).view(torch.uint32)
        t[pre + name + ".scales"] = torch.full((rows, d // 64), 0.002).bfloat16()
        t[pre + name + ".biases"] = torch.full((rows, d // 64), -0.25).bfloat16()
        q[pre + name] = {"group_size": 64, "bits": 8}
    st.save_file(t, str(path / "model.safetensors"), metadata={"format": "mlx"})
    (path / "config.json").write_text(json.dumps(
        {"quantization": q, "text_config": {"num_experts_per_tok": 4}}))
    return t, pre


def test_loader_reads_mxfp4(pkg, tmp_path):
    t, pre = write_checkpoint(tmp_path)
    b = pkg.loader.qwen35_moe_block(tmp_path, 2, "cpu")
    up = b.switch_mlp.up_proj
    assert (up.mode, up.group_size, up.bits, up.biases) == ("mxfp4", 32, 4, None)
    assert torch.equal(up.weight.view(torch.uint32), t[pre + "switch_mlp.up_proj.weight"])
    assert torch.equal(up.scales, t[pre + "switch_mlp.up_proj.scales"])
    down = b.shared_expert.down_proj
    assert down.mode == "mxfp4" and down.scales.shape == (1, 256, 4)
    assert b.gate_weight.mode == "affine" and b.gate_weight.bits == 8
    (tmp_path / "other").mkdir()
    write_checkpoint(tmp_path / "other", mode="nvfp4")
    with pytest.raises(pkg.MlxrMoeError, match="mode"):
        pkg.loader.qwen35_moe_block(tmp_path / "other", 2, "cpu")


@gpu
@pytest.mark.parametrize("T", [1, 300])
def test_loaded_block_runs(pkg, dev, tmp_path, T):
    """The loaded block against its own modules: the expert rows combined
    in the bf16 chain of a quantised router."""
    write_checkpoint(tmp_path)
    b = pkg.loader.qwen35_moe_block(tmp_path, 2, dev)
    x = torch.randn((T, 256), generator=torch.Generator().manual_seed(T)).bfloat16().to(dev)
    out = b.forward(x)
    assert out.dtype == torch.bfloat16
    idx, w = pkg.ops.router_topk_quantized(x, b.gate_weight, 4)
    assert torch.equal(b.last_indices, idx)
    y = b.switch_mlp.forward(x, idx).double()
    sy = b.shared_expert.forward(x).double()
    sg = b.shared_expert_gate_weight
    sg = pkg.ops.dequantize(sg.weight[0], sg.scales[0], sg.biases[0], 64, 8, torch.float32)
    gate = torch.sigmoid(x.double() @ sg.double().t())
    ref = (y * w.double()[:, :, None]).sum(1) + sy * gate
    mass = (y * w.double()[:, :, None]).abs().sum(1) + (sy * gate).abs()
    # each row and product, the sums and the gate rounded to bf16: four steps
    assert bool(((out.double() - ref).abs() <= 4 * 2.0 ** -7 * mass).all())


# ------------------------------------------------------ quantise, dequantise
@gpu
def test_every_code_and_scale(pkg, dev):
    """All 16 codes under all 256 scale bytes, to f32 and bf16."""
    code = torch.arange(32) % 16
    words = sum(code.view(4, 8)[:, i] << (4 * i) for i in range(8))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    wq = words.repeat(256, 1).contiguous()
    sc = torch.arange(256).to(torch.uint8)[:, None]
    want = values64(wq, sc)
    for dt in (torch.float32, torch.bfloat16):
        got = pkg.ops.dequantize(wq.to(dev), sc.to(dev), mode="mxfp4", out_dtype=dt).cpu()
        ref = want.to(dt)  # exact, or an infinity past the type's range
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        ok = ~torch.isnan(ref)
        assert torch.equal(got[ok], ref[ok])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (2, 5, 96), (7, 2048), (1, 509, 2080)])
def test_quantise_is_nearest(pkg, dev, dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    w = (torch.randn(shape, generator=g) * 0.02).to(dtype)
    w.view(-1)[:32] = 0.0  # a group of zeros
    wq, sc, bi = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    assert bi is None and wq.shape == shape[:-1] + (shape[-1] // 8,)
    want, byte = quantise64(w)
    assert torch.equal(sc.cpu().long(), byte)
    assert torch.equal(values64(wq, sc), want)
    back = pkg.ops.dequantize(wq, sc, mode="mxfp4", out_dtype=dtype)
    assert torch.equal(back.cpu().double(), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_borders_and_extremes(pkg, dev, dtype):
    """Midpoints between neighbours, magnitudes past 6, subnormal groups,
    groups with one large value, infinities and NaN."""
    rows = []
    for scale in (1.0, 2.0 ** -20, 2.0 ** 100, 2.0 ** -118):
        mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9375])
        near = torch.cat([mid, mid * (1 + 2 ** -7), mid * (1 - 2 ** -7)])
        rows.append(torch.cat([near * scale, torch.tensor([4.0, -6.0]) * scale]))
    tiny = torch.arange(32) * 2.0 ** -130
    rows += [tiny, -tiny, torch.arange(32) * 2.0 ** -127, torch.full((32,), 2.0 ** -126)]
    one = torch.zeros(32)
    one[17] = 3.0e38
    rows.append(one)
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.ones(32)
        r[5] = bad
        rows.append(r)
    w = torch.stack(rows).to(dtype)
    wq, sc, _ = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    want, byte = quantise64(w)
    assert torch.equal(sc.cpu().long(), byte)
    got = values64(wq, sc)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok])
    assert bool((wq.cpu()[-3:] == 0).all())  # a bad group's codes


@gpu
@pytest.mark.parametrize("dtype,rows", [(torch.bfloat16, 65601), (torch.float32, 33003)])
def test_quantise_larger_than_the_caches(pkg, dev, dtype, rows):
    """An array past 256 MB: the same codes, scales and values as its parts."""
    g = torch.Generator(device=dev).manual_seed(5)
    w = torch.randn((rows, 2080), generator=g, device=dev).to(dtype)
    assert w.numel() * w.element_size() > 2 ** 28
    wq, sc, _ = pkg.ops.quantize(w, mode="mxfp4")
    v = pkg.ops.dequantize(wq, sc, mode="mxfp4", out_dtype=dtype)
    for a, b in ((0, 1), (1, rows // 2), (rows // 2, rows)):
        q, s, _ = pkg.ops.quantize(w[a:b], mode="mxfp4")
        assert torch.equal(q, wq[a:b]) and torch.equal(s, sc[a:b])
        assert torch.equal(pkg.ops.dequantize(q, s, mode="mxfp4", out_dtype=dtype), v[a:b])


@gpu
def test_quantise_strided_and_unaligned(pkg, dev):
    w = torch.randn(6, 128, device=dev)
    q = pkg.ops.quantize
    a = q(w[::2, 64:], mode="mxfp4")
    b = q(w[::2, 64:].contiguous(), mode="mxfp4")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for dt in (torch.float32, torch.bfloat16):
        flat = torch.randn(1 + 64 * 3, device=dev).to(dt)
        v = flat[1:].view(3, 64)  # not 16-byte aligned
        a, b = q(v, mode="mxfp4"), q(v.clone(), mode="mxfp4")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------- product
def gather_case(pkg, dev, E, N, K, idx, x, seed=0, lhs=None, wq_sc=None):
    g = torch.Generator().manual_seed(seed)
    wq, sc = wq_sc if wq_sc is not None else bank(g, (E, N, K))
    kw = {"lhs_indices": lhs.to(dev)} if lhs is not None else {}
    y = pkg.ops.gather_qmm(x.to(dev), wq.to(dev), sc.to(dev), rhs_indices=idx.to(dev),
                           mode="mxfp4", **kw).cpu()
    return y, wq, sc


@gpu
@pytest.mark.parametrize("K", [64, 128, 192, 320, 768, 2048, 4096])
@pytest.mark.parametrize("T,topk", [(1, 1), (1, 8), (3, 2), (9, 8), (40, 4)])
def test_gather_few_rows(pkg, dev, K, T, topk):
    """Work items: one row, a few, more than one item per expert; input dims
    that end inside a step; one 64-channel tile and several."""
    E, N = 11, 64 if K % 128 else 192
    g = torch.Generator().manual_seed(K + T)
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = torch.randint(0, E, (T, topk), generator=g, dtype=torch.int32)
    idx[T // 2:] = idx[T // 2, 0]  # crowd one expert, the same one several times a row
    y, wq, sc = gather_case(pkg, dev, E, N, K, idx, x, K)
    w64 = values64(wq, sc)
    for e in idx.unique().tolist():
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(y[t, k, 0], x[t, 0, 0].double(), w64[e], K)


@gpu
@pytest.mark.parametrize("E,N,K,T,topk,skew", [
    (4, 64, 64, 300, 2, 0),        # one N-tile, one x stage
    (8, 192, 192, 200, 4, 0),      # part of a line, part of an N-tile
    (8, 320, 768, 150, 4, 1),      # skewed: one expert takes most rows
    (16, 768, 2048, 130, 4, 0),    # 64-row tiles
    (3, 256, 512, 333, 2, 0),      # 128-row tiles, a ragged last one
    (5, 448, 4096, 70, 8, 0),      # the largest input dim
    (2, 64, 320, 777, 1, 1),
])
def test_gather_many_rows(pkg, dev, E, N, K, T, topk, skew):
    g = torch.Generator().manual_seed(E * N + K)
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = torch.randint(0, E, (T, topk), generator=g, dtype=torch.int32)
    if skew:
        idx[: T * 3 // 4] = 1
    assert pkg.ops.gather_qmm_tiled(T * topk, E)  # past the rule for tiles
    y, wq, sc = gather_case(pkg, dev, E, N, K, idx, x, K)
    w64 = values64(wq, sc)
    for e in idx.unique().tolist():
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(y[t, k, 0], x[t, 0, 0].double(), w64[e], K)


@gpu
@pytest.mark.parametrize("E,N,K,T,topk", [
    (128, 64, 64, 95, 2),       # just under the tiles' rule
    (128, 64, 64, 96, 2),       # just on it: 1.5 rows an expert
    (130, 192, 192, 65, 3),     # part of a line, part of an N-tile
    (128, 320, 768, 300, 4),    # several tiles for the crowded experts
    (140, 64, 4096, 200, 5),    # the largest input dim
    (200, 256, 2048, 1200, 3),  # 18 rows an expert
])
def test_gather_short_tiles(pkg, dev, E, N, K, T, topk):
    """Many experts with few rows each, some just at and past a tile's end."""
    g = torch.Generator().manual_seed(E * T + K)
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = torch.randint(7, E, (T, topk), generator=g, dtype=torch.int32)
    at = 0
    for e, rows in enumerate([32, 33, 31, 1]):  # as many as there are rows for
        take = idx.view(-1)[at:at + rows]
        take.fill_(e)
        at += len(take)
    y, wq, sc = gather_case(pkg, dev, E, N, K, idx, x, K)
    w64 = values64(wq, sc)
    for e in idx.unique().tolist():
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(y[t, k, 0], x[t, 0, 0].double(), w64[e], K)


@gpu
@pytest.mark.parametrize("T", [5, 400])
def test_gather_lhs_M_and_bad_indices(pkg, dev, T):
    """lhs indices, several rows per batch, and indices out of range: their
    rows are zero, the status word says so, the others are as without them."""
    E, N, K, M = 6, 128, 256, 2
    g = torch.Generator().manual_seed(T)
    x = torch.randn((7, M, K), generator=g).bfloat16()
    rhs = torch.randint(0, E, (T,), generator=g, dtype=torch.int32)
    lhs = torch.randint(0, 7, (T,), generator=g, dtype=torch.int32)
    rhs[2], lhs[4] = E, 7
    rhs[3] = -1
    wq, sc = bank(g, (E, N, K))
    out = pkg.ops.gather_qmm(x.to(dev), wq.to(dev), sc.to(dev), lhs_indices=lhs.to(dev),
                             rhs_indices=rhs.to(dev), mode="mxfp4")
    assert pkg.ops.workspace_status(out._mlxr_workspace) == 1
    y = out.cpu()
    assert bool((y[2:5] == 0).all())
    w64 = values64(wq, sc)
    for b in range(T):
        if b not in (2, 3, 4):
            check_sum(y[b], x[lhs[b]].double(), w64[rhs[b]], K)


@gpu
@pytest.mark.parametrize("n", [1, 8, 63, 64, 65, 130])
@pytest.mark.parametrize("kind", ["one", "all", "pairs", "bad"])
def test_gather_groups_of_rows(pkg, dev, n, kind):
    """Around the 64 rows that the streaming kernel groups by itself: every row
    the same expert (items of 8), every row its own, runs of two, and no row
    with an expert at all."""
    E, N, K = 140, 64, 192
    g = torch.Generator().manual_seed(n)
    wq, sc = bank(g, (E, N, K))
    x = torch.randn((n, 1, K), generator=g).bfloat16()
    idx = {"one": torch.full((n,), 3), "all": torch.arange(n).flip(0),
           "pairs": torch.arange(n) // 2 + 1, "bad": torch.full((n,), E + 5)}[kind]
    y = pkg.ops.gather_qmm(x.to(dev), wq.to(dev), sc.to(dev), rhs_indices=idx.int().to(dev),
                           mode="mxfp4")
    status = pkg.ops.workspace_status(y._mlxr_workspace)
    y = y.cpu()
    if kind == "bad":
        assert status == 1 and bool((y == 0).all())
        return
    assert status == 0
    w64 = values64(wq, sc)
    for e in idx.unique().tolist():
        r = (idx == e).nonzero()[:, 0]
        check_sum(y[r, 0], x[r, 0].double(), w64[e], K)


@gpu
@pytest.mark.parametrize("T,topk,E", [(40, 16, 8), (520, 1, 2), (3000, 2, 3), (33000, 1, 5),
                                      (600, 3, 1024)])
def test_gather_sorts(pkg, dev, T, topk, E):
    """The tiles' own sort: few rows to more than it takes (then the general
    dispatch), indices out of range among them, an expert without rows."""
    N, K = 64, 64
    g = torch.Generator().manual_seed(T)
    wq, sc = bank(g, (E, N, K))
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = torch.randint(0, E - 1, (T, topk), generator=g, dtype=torch.int32)
    idx[T // 3, 0], idx[T // 2, topk - 1] = E, -1
    y = pkg.ops.gather_qmm(x.to(dev), wq.to(dev), sc.to(dev), rhs_indices=idx.to(dev),
                           mode="mxfp4")
    assert pkg.ops.workspace_status(y._mlxr_workspace) == 1
    y, w64 = y.cpu(), values64(wq, sc)
    assert bool((y[(idx < 0) | (idx >= E)] == 0).all())
    for e in range(E - 1):
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(y[t, k, 0], x[t, 0, 0].double(), w64[e], K)


@gpu
@pytest.mark.parametrize("T,topk", [(3, 2), (800, 2)])
def test_gather_weights_past_32_bits(pkg, dev, T, topk):
    """8.6 GB of codes in one tensor: the last experts' rows, from the
    streaming kernel and from tiles."""
    E, N, K = 1024, 4096, 4096
    g = torch.Generator(device=dev).manual_seed(1)
    wq = torch.randint(-2 ** 31, 2 ** 31 - 1, (E, N, K // 8), generator=g, device=dev,
                       dtype=torch.int32)
    sc = torch.randint(118, 122, (E, N, K // 32), generator=g, device=dev, dtype=torch.uint8)
    idx = torch.randint(0, E, (T, topk), generator=g, device=dev, dtype=torch.int32)
    idx[0, 0], idx[1, 1], idx[2, 0] = E - 1, E - 2, 513
    x = torch.randn((T, 1, 1, K), generator=g, device=dev).bfloat16()
    y = pkg.ops.gather_qmm(x, wq, sc, rhs_indices=idx, mode="mxfp4").cpu()
    x, idx = x.cpu().double(), idx.cpu()
    for e in (E - 1, E - 2, 513):
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(y[t, k, 0], x[t, 0, 0], values64(wq[e:e + 1].cpu(), sc[e:e + 1].cpu())[0], K)


@gpu
@pytest.mark.parametrize("T", [3, 600])
def test_ffn_leaves_rows_of_bad_indices_out(pkg, dev, T):
    """-1 leaves a row out silently, another bad index sets the status word;
    the other rows are as without them."""
    w, x, idx = ffn_inputs(5, 8, 128, 64, T, 4)
    m = ffn(pkg, dev, w)
    a = m.forward(x.to(dev), idx.to(dev)).cpu()
    assert pkg.ops.workspace_status(m.last_workspace) == 0
    cut = idx.clone()
    cut[1, 2] = -1
    b = m.forward(x.to(dev), cut.to(dev)).cpu()
    assert pkg.ops.workspace_status(m.last_workspace) == 0
    cut[2, 0] = 8
    c = m.forward(x.to(dev), cut.to(dev)).cpu()
    assert pkg.ops.workspace_status(m.last_workspace) == 1
    keep = torch.ones((T, 4), dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(a[keep], b[keep])
    keep[2, 0] = False
    assert torch.equal(a[keep], c[keep])


@gpu
@pytest.mark.parametrize("T", [2, 600])
def test_gather_extreme_scales(pkg, dev, T):
    """Scale bytes at both ends of the range, NaN scales, infinities in x."""
    E, N, K = 2, 64, 128
    g = torch.Generator().manual_seed(T)
    wq, sc = bank(g, (E, N, K))
    sc[0, :, 0] = 0        # 2^-127: subnormal weights
    sc[0, 5, 1] = 255      # a NaN group: channel 5 of expert 0
    sc[1, :, :] = 120
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = (torch.arange(T, dtype=torch.int32) % 2)[:, None]
    y, _, _ = gather_case(pkg, dev, E, N, K, idx, x, wq_sc=(wq, sc))
    w64 = values64(wq, sc)
    keep = torch.arange(N) != 5
    assert bool(torch.isnan(y[0::2, 0, 0, 5]).all())
    check_sum(y[0::2, 0, 0][:, keep], x[0::2, 0, 0].double(), w64[0][keep], K)
    check_sum(y[1::2, 0, 0], x[1::2, 0, 0].double(), w64[1], K)
    # the largest scales that stay finite in the sums
    sc[1, :, :] = 250
    y, _, _ = gather_case(pkg, dev, E, N, K, idx, x * 2.0 ** -60, wq_sc=(wq, sc))
    check_sum(y[1::2, 0, 0], (x * 2.0 ** -60)[1::2, 0, 0].double(), values64(wq, sc)[1], K)
    # an infinity in one row leaves the others as they are
    x2 = x.clone()
    x2[1, 0, 0, 3] = float("inf")
    sc[1, :, :] = 120
    a, _, _ = gather_case(pkg, dev, E, N, K, idx, x, wq_sc=(wq, sc))
    b, _, _ = gather_case(pkg, dev, E, N, K, idx, x2, wq_sc=(wq, sc))
    rest = torch.arange(T) != 1
    same = (a[rest] == b[rest]) | (torch.isnan(a[rest]) & torch.isnan(b[rest]))
    assert bool(same.all())
    code3 = (wq[1, :, 0].long() >> 12) & 7  # input 3's codes: inf * 0 is NaN
    assert bool((torch.isnan(b[1, 0, 0]) == (code3 == 0)).all())


@gpu
def test_gather_empty(pkg, dev):
    wq, sc = bank(torch.Generator().manual_seed(0), (2, 64, 64))
    y = pkg.ops.gather_qmm(torch.zeros((1, 1, 64), dtype=torch.bfloat16, device=dev), wq.to(dev),
                           sc.to(dev), rhs_indices=torch.zeros(0, dtype=torch.int32, device=dev),
                           mode="mxfp4")
    assert y.shape == (0, 1, 64)


@gpu
@pytest.mark.parametrize("T", [6, 700])
def test_gather_scales_at_any_address(pkg, dev, T):
    """Scales at an address that the kernels do not take (a view one byte into
    its storage) are copied."""
    E, N, K = 3, 128, 320
    g = torch.Generator().manual_seed(T)
    wq, sc = bank(g, (E, N, K))
    x = torch.randn((T, 1, 1, K), generator=g).bfloat16()
    idx = torch.randint(0, E, (T, 1), generator=g, dtype=torch.int32)
    a, _, _ = gather_case(pkg, dev, E, N, K, idx, x, wq_sc=(wq, sc))
    store = torch.zeros(sc.numel() + 1, dtype=torch.uint8, device=dev)
    store[1:] = sc.flatten().to(dev)
    b = pkg.ops.gather_qmm(x.to(dev), wq.to(dev), store[1:].view(sc.shape),
                           rhs_indices=idx.to(dev), mode="mxfp4").cpu()
    assert torch.equal(a, b)


# ------------------------------------------------------------------- modules
def glu64(x, w, idx, act):
    """Expert outputs in 64 bits (nothing rounded between), and the bound of
    each one's distance: gate and up are f32 sums of d products; the
    activation's derivative is at most 1.13 u and g, its f32 evaluation a few
    steps off; h is rounded to bf16 once, y is an f32 sum of f products and
    rounded once."""
    T, K = idx.shape
    d, f = x.shape[1], w[2].shape[2]
    y = torch.zeros((T, K, w[2].shape[1]), dtype=torch.float64)
    bound = torch.zeros_like(y)
    for e in idx.unique().tolist():
        t, k = (idx == e).nonzero(as_tuple=True)
        g, u = x[t] @ w[0][e].t(), x[t] @ w[1][e].t()
        eg, eu = (d * 2.0 ** -23 * (x[t].abs() @ m[e].abs().t()) for m in w[:2])
        if act == "swiglu":
            h = g * torch.sigmoid(g) * u
        else:  # with the constants of the reference's bf16 chain
            c, s = 0.044677734375, 0.796875
            h = 0.5 * g * (1.0 + torch.tanh(s * (g + c * g ** 3))) * u
        eh = 1.13 * u.abs() * eg + g.abs() * eu + 2.0 ** -19 * (h.abs() + (g * u).abs())
        eh = eh + 2.0 ** -8 * (h.abs() + eh)
        wd = w[2][e].abs().t()
        y[t, k] = h @ w[2][e].t()
        err = eh @ wd + f * 2.0 ** -23 * ((h.abs() + eh) @ wd)
        bound[t, k] = err + 2.0 ** -8 * (y[t, k].abs() + err)
    return y, bound


def ffn_inputs(seed, E, d, f, T, K):
    g = torch.Generator().manual_seed(seed)
    w = [bank(g, s) for s in ((E, f, d), (E, f, d), (E, d, f))]
    x = torch.randn((T, d), generator=g).bfloat16()
    idx = torch.rand((T, E), generator=g).topk(K, dim=1).indices.to(torch.int32)
    return w, x, idx


def ffn(pkg, dev, w):
    nn = pkg.nn
    return nn.SplitSwitchFfn(*[
        nn.QuantizedSwitchLinear(q.to(dev), s.to(dev), mode="mxfp4") for q, s in w])


@gpu
@pytest.mark.parametrize("E,d,f,T,K", [(16, 256, 128, 1, 4), (16, 256, 192, 7, 4),
                                       (32, 512, 256, 30, 8), (8, 2048, 320, 33, 2),
                                       (16, 256, 128, 300, 4), (8, 512, 192, 600, 2)])
def test_split_ffn(pkg, dev, E, d, f, T, K):
    """One token to M-tiles: forward, forward_with_combine, and the same
    results from the three projections one by one."""
    w, x, idx = ffn_inputs(T + d, E, d, f, T, K)
    m = ffn(pkg, dev, w)
    y = m.forward(x.to(dev), idx.to(dev))
    want, bound = glu64(x.double(), [values64(*b) for b in w], idx, "swiglu")
    err = (y.cpu().double() - want).abs()
    assert bool((err <= bound).all())
    # two independent roundings (h and y), each 2^-8 / sqrt(3) of its value in the
    # root mean square at most
    assert float(err.norm() / want.norm()) < 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5
    wts = torch.rand((T, K), generator=torch.Generator().manual_seed(1)).to(dev)
    out = m.forward_with_combine(x.to(dev), idx.to(dev), wts)
    ref = (y.double() * wts.double()[:, :, None]).sum(1)
    mass = (y.double() * wts.double()[:, :, None]).abs().sum(1)
    assert bool(((out.double() - ref).abs() <= 2 * K * 2.0 ** -24 * mass).all())
    g = m.gate_proj.apply(x.to(dev)[:, None, None, :], idx.to(dev))[:, :, 0]
    gw = values64(*w[0])
    for e in idx.unique().tolist():
        t, k = (idx == e).nonzero(as_tuple=True)
        check_sum(g.cpu()[t, k], x[t].double(), gw[e], d)


@gpu
@pytest.mark.parametrize("dtype", [torch.int16, torch.uint8, torch.int64])
def test_split_ffn_takes_any_integer_indices(pkg, dev, dtype):
    w, x, idx = ffn_inputs(2, 8, 256, 128, 5, 4)
    m = ffn(pkg, dev, w)
    want = m.forward(x.to(dev), idx.to(dev))
    assert torch.equal(m.forward(x.to(dev), idx.to(dtype).to(dev)), want)
    # (a transposed tensor of them too)
    t = idx.to(dtype).to(dev).t().contiguous().t()
    assert torch.equal(m.forward(x.to(dev), t), want)


@gpu
@pytest.mark.parametrize("T", [1, 9, 260])
@pytest.mark.parametrize("act", ["geglu", "swiglu"])
def test_packed_ffn(pkg, dev, T, act):
    E, d, f, K = 8, 256, 128, 4
    w, x, idx = ffn_inputs(T, E, d, f, T, K)
    gu = (torch.cat([w[0][0], w[1][0]], 1), torch.cat([w[0][1], w[1][1]], 1))
    nn = pkg.nn
    lin = lambda b: nn.QuantizedSwitchLinear(b[0].to(dev), b[1].to(dev), mode="mxfp4")  # noqa: E731
    m = nn.PackedSwitchFfn(lin(gu), lin(w[2]), act)
    y = m.forward(x.to(dev), idx.to(dev)).cpu().double()
    want, bound = glu64(x.double(), [values64(*b) for b in w], idx, act)
    assert bool(((y - want).abs() <= bound).all())
    if act == "swiglu":  # the packed tensor is the split ones, row for row
        assert torch.equal(y, ffn(pkg, dev, w).forward(x.to(dev), idx.to(dev)).cpu().double())


@gpu
@pytest.mark.parametrize("T", [1, 5, 90, 300])
@pytest.mark.parametrize("shared_mx", [True, False])
def test_block(pkg, dev, T, shared_mx):
    """The block over mxfp4 experts, its shared expert in the same form (in
    the same launches) or affine: routing, shared branch and combine as with
    the expert outputs of the modules alone; and the residual form."""
    E, d, f, K = 16, 256, 128, 4
    nn, ops = pkg.nn, pkg.ops
    w, x, _ = ffn_inputs(T, E, d, f, T, K)
    g = torch.Generator().manual_seed(7)
    gate_w = torch.randn((E, d), generator=g).to(dev) * 0.1
    sg = torch.randn((1, d), generator=g).to(dev) * 0.1
    dense = [(torch.randn(s, generator=g) * 0.05).bfloat16().to(dev)
             for s in ((f, d), (f, d), (d, f))]
    mode = "mxfp4" if shared_mx else "affine"
    shared = nn.SwigluMlp(*[nn.QuantizedLinear.try_from_linear(v, mode=mode) for v in dense])
    m = ffn(pkg, dev, w)
    blk = nn.Qwen35MoeBlock(gate_w, m, K, shared, sg)
    xd = x.to(dev)
    out = blk.forward(xd)
    idx, wts = ops.router_topk(xd, gate_w, K)
    y = m.forward(xd, idx)
    sy = shared.forward(xd)
    logit = xd.float() @ sg[0]
    assert torch.equal(blk.last_indices, idx)
    ref = (y.double() * wts.double()[:, :, None]).sum(1)
    sgate = torch.sigmoid(logit.double())[:, None]
    ref = ref + sy.double() * sgate
    mass = (y.double() * wts.double()[:, :, None]).abs().sum(1) + (sy.double() * sgate).abs()
    # the folded rows may be summed in another slicing of the input dim: a bf16
    # step of any y; the shared gate's logit an f32 sum of d terms
    lerr = d * 2.0 ** -22 * (xd.double().abs() @ sg[0].double().abs())[:, None]
    tol = mass * (2.0 ** -6 + lerr)
    assert bool(((out.double() - ref).abs() <= tol).all())
    if T <= 5:
        n = nn.RmsNorm(torch.ones(d).to(dev))
        h = blk.forward_residual(xd, n)
        assert bool(torch.isfinite(h).all())
        assert torch.allclose(h, xd.float() + blk.forward(n.forward(xd)), rtol=1e-5, atol=1e-5)


@gpu
@pytest.mark.parametrize("T", [70, 300])
def test_block_many_experts(pkg, dev, T):
    """Short tiles from the block's own dispatch, the shared expert's rows in
    the same launches, and the same block without a workspace of its own."""
    E, d, f, K = 128, 256, 192, 4
    nn, ops = pkg.nn, pkg.ops
    w, x, _ = ffn_inputs(T, E, d, f, T, K)
    g = torch.Generator().manual_seed(8)
    gate_w = torch.randn((E, d), generator=g).to(dev) * 0.1
    sg = torch.randn((1, d), generator=g).to(dev) * 0.1
    dense = [(torch.randn(s, generator=g) * 0.05).bfloat16().to(dev)
             for s in ((f, d), (f, d), (d, f))]
    shared = nn.SwigluMlp(*[nn.QuantizedLinear.try_from_linear(v, mode="mxfp4") for v in dense])
    m = ffn(pkg, dev, w)
    blk = nn.Qwen35MoeBlock(gate_w, m, K, shared, sg)
    xd = x.to(dev)
    out = blk.forward(xd)
    idx, wts = ops.router_topk(xd, gate_w, K)
    y, sy = m.forward(xd, idx), shared.forward(xd)
    sgate = torch.sigmoid((xd.float() @ sg[0]).double())[:, None]
    terms = y.double() * wts.double()[:, :, None]
    mass = terms.abs().sum(1) + (sy.double() * sgate).abs()
    lerr = d * 2.0 ** -22 * (xd.double().abs() @ sg[0].double().abs())[:, None]
    # (as test_block: the folded rows may take another slicing, a bf16 step of any y)
    assert bool(((out.double() - terms.sum(1) - sy.double() * sgate).abs()
                 <= mass * (2.0 ** -6 + lerr)).all())
    C = pkg._capi
    bare = torch.empty_like(out)
    stream = torch.cuda.current_stream().cuda_stream
    C.check(C.lib().mlxr_moe_block_forward_noalloc(
        ctypes.byref(blk.descriptor()), xd.data_ptr(), T, bare.data_ptr(), None, None, stream))
    assert torch.equal(bare, out)


@gpu
@pytest.mark.parametrize("T", [3, 400])
def test_graph_and_streams(pkg, dev, T):
    """A captured pass replayed with eager work between, and the same pass on
    a side stream: the eager results, bit for bit."""
    w, x, idx = ffn_inputs(3, 8, 256, 128, T, 4)
    m = ffn(pkg, dev, w)
    xs, ids = x.to(dev), idx.to(dev)
    wq, sc = m.gate_proj.weight, m.gate_proj.scales

    def step():
        y = m.forward(xs, ids)
        g = pkg.ops.gather_qmm(xs[:, None, None, :], wq, sc, rhs_indices=ids, mode="mxfp4")
        q = pkg.ops.quantize(y, mode="mxfp4")
        return [y, g, pkg.ops.dequantize(q[0], q[1], mode="mxfp4")]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        xs.copy_((x + i).bfloat16())
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


def test_optional_int_reads_its_argument_at_every_call(pkg):
    """Anything int() takes, and its value now, whatever a call before held."""
    import numpy as np
    of = pkg._capi.OptionalInt.of
    t = torch.tensor(64)
    assert of(t).value == 64
    t.fill_(32)
    assert of(t).value == 32
    assert of(np.array(8)).value == 8 and of(np.int64(4)).value == 4 and of(4.0).value == 4
    o = of(5)
    o.value = 6  # the caller's own
    assert of(5).value == 5 and of(None).has_value == 0 and of(5).has_value == 1


@pytest.mark.parametrize("named", [{}, {"mode": None}, {"mode": "affine"}])
def test_loader_takes_a_mode_that_says_nothing(pkg, named):
    """A mode of null, in the body or in an override, is none: affine."""
    pre = "model.layers.0.mlp.gate"
    q = pkg.loader.QuantizationConfig({"group_size": 64, "bits": 4, **named,
                                       pre: {"group_size": 64, "bits": 8, **named}})
    assert q.mode_for_path(pre) == "affine" and q.mode_for_path("other") == "affine"
    assert q.for_path(pre) == (64, 8)


@gpu
@pytest.mark.parametrize("T", [5, 600])
def test_indices_past_32_bits(pkg, dev, T):
    """64-bit indices that no 32-bit one holds are out of range, in the plain
    product (rows cleared) and in the modules (rows left out)."""
    w, x, idx = ffn_inputs(6, 8, 128, 64, T, 4)
    wide, ok = idx.long(), torch.ones((T, 4), dtype=torch.bool)
    wide[0, 1], wide[2, 3], wide[3, 0] = 2 ** 32 + 1, 2 ** 31, -2 ** 32 + 2
    ok[0, 1] = ok[2, 3] = ok[3, 0] = False
    m, xd = ffn(pkg, dev, w), x.to(dev)
    up = m.up_proj
    kw = {"rhs_indices": wide.to(dev), "mode": "mxfp4"}
    y = pkg.ops.gather_qmm(xd[:, None, None, :], up.weight, up.scales, **kw)
    assert pkg.ops.workspace_status(y._mlxr_workspace) == 1
    kw["rhs_indices"] = idx.to(dev)
    want = pkg.ops.gather_qmm(xd[:, None, None, :], up.weight, up.scales, **kw)
    assert torch.equal(y[ok], want[ok]) and bool((y[~ok] == 0).all())
    gu = [torch.cat([w[0][i], w[1][i]], 1).to(dev) for i in (0, 1)]
    packed = pkg.nn.PackedSwitchFfn(pkg.nn.QuantizedSwitchLinear(*gu, mode="mxfp4"), m.down_proj,
                                    "swiglu")
    for mod in (m, packed):
        a = mod.forward(xd, idx.to(dev))
        assert pkg.ops.workspace_status(mod.last_workspace) == 0
        b = mod.forward(xd, wide.to(dev))
        assert pkg.ops.workspace_status(mod.last_workspace) == 1
        assert torch.equal(a[ok], b[ok])


def test_rule_for_tiles(pkg):
    """Which kernel a product of mxfp4 experts takes (host logic, no GPU): tiles
    from 1.5 rows an expert, and with fewer than 128 experts from 16 rows an expert or 320
    in all, with fewer than 8 from 512; the affine rule beside it is its own."""
    q, mx = pkg.ops.gather_qmm_tiled, "mxfp4"
    assert not q(191, 128, mx) and q(192, 128, mx)
    assert not q(1535, 1024, mx) and q(1536, 1024, mx)
    assert not q(127, 8, mx) and q(128, 8, mx)
    assert not q(319, 127, mx) and q(320, 127, mx)
    assert not q(511, 7, mx) and q(512, 7, mx)
    assert not q(511, 1, mx) and q(512, 1, mx)
    assert not q(0, 8, mx)
    for rows, experts in ((192, 128), (1536, 1024), (512, 1), (511, 1), (6000, 128)):
        assert q(rows, experts) == q(rows, experts, "affine")
    assert not q(192, 128) and q(6000, 128)
    with pytest.raises(pkg.MlxrMoeError, match="negative"):
        q(-1, 8, mx)
    with pytest.raises(pkg.MlxrMoeError, match="mode"):
        q(1, 8, "nvfp4")
    f = pkg._capi.lib().mlxr_moe_gather_qmm_tiled_mode
    assert f(192, 128, b"mxfp4") == 1 and f(192, 128, b"affine") == 0 and f(192, 128, None) == 0
    assert f(192, -1, b"mxfp4") == -1 and f(192, 128, b"nvfp4") == -1


def test_rule_of_the_tested_sizes(pkg):
    """The products above that are meant to run as tiles do, and those meant to
    stay just under the rule do."""
    q = pkg.ops.gather_qmm_tiled
    for E, rows in ((4, 600), (8, 800), (8, 600), (16, 520), (3, 666), (5, 560), (2, 777),
                    (128, 192), (130, 195), (128, 1200), (140, 1000), (200, 3600),
                    (8, 640), (2, 520), (3, 6000), (5, 33000), (1024, 1800), (1024, 1600)):
        assert q(rows, E, "mxfp4"), (E, rows)
    for E, rows in ((11, 1), (11, 8), (11, 6), (11, 72), (11, 160), (128, 190), (140, 130)):
        assert not q(rows, E, "mxfp4"), (E, rows)


@gpu
@pytest.mark.parametrize("E,f,T,K,tiled", [
    (8, 128, 1, 2, False),    # the input dim in four slices
    (4, 1024, 20, 2, False),  # two
    (4, 1024, 80, 2, False),  # one, over 64 rows: items from a dispatch
    (8, 192, 70, 2, True),    # 32-row tiles
    (8, 192, 130, 2, True),   # 64-row tiles
    (8, 192, 300, 2, True),   # 128-row tiles
])
def test_split_ffn_widest_input(pkg, dev, E, f, T, K, tiled):
    """Gate and up over 4096 inputs, the most there are, in every form."""
    d = 4096
    w, x, idx = ffn_inputs(T + f, E, d, f, T, K)
    assert pkg.ops.gather_qmm_tiled(T * K, E, "mxfp4") == tiled
    m = ffn(pkg, dev, w)
    want, bound = glu64(x.double(), [values64(*b) for b in w], idx, "swiglu")
    y = m.forward(x.to(dev), idx.to(dev))
    assert bool(((y.cpu().double() - want).abs() <= bound).all())
    assert torch.equal(m.forward(x.to(dev), idx.to(dev)), y)


@gpu
@pytest.mark.parametrize("T", [9, 300])
def test_packed_geglu_widest_input(pkg, dev, T):
    E, d, f, K = 8, 4096, 128, 4
    w, x, idx = ffn_inputs(T, E, d, f, T, K)
    lin = lambda b: pkg.nn.QuantizedSwitchLinear(b[0].to(dev), b[1].to(dev), mode="mxfp4")  # noqa: E731
    gu = (torch.cat([w[0][0], w[1][0]], 1), torch.cat([w[0][1], w[1][1]], 1))
    y = pkg.nn.PackedSwitchFfn(lin(gu), lin(w[2]), "geglu").forward(x.to(dev), idx.to(dev))
    want, bound = glu64(x.double(), [values64(*b) for b in w], idx, "geglu")
    assert bool(((y.cpu().double() - want).abs() <= bound).all())


def shared_inputs(T, d, f):
    w, x, _ = ffn_inputs(T, 1, d, f, T, 1)
    idx = torch.zeros((T, 1), dtype=torch.int32)
    return w, x, glu64(x.double(), [values64(*b) for b in w], idx, "swiglu")


def shared_mlp(pkg, dev, w):
    return pkg.nn.SwigluMlp(*[pkg.nn.QuantizedLinear(q[0].to(dev), s[0].to(dev), mode="mxfp4")
                              for q, s in w])


@gpu
@pytest.mark.parametrize("d,f", [(256, 192), (4096, 64)])
@pytest.mark.parametrize("T", [1, 511, 512, 650])
def test_one_expert(pkg, dev, T, d, f):
    """SwigluMlp alone, just under the rule for tiles, on it and past it with a
    ragged last tile."""
    w, x, (want, bound) = shared_inputs(T, d, f)
    assert pkg.ops.gather_qmm_tiled(T, 1, "mxfp4") == (T >= 512)
    y = shared_mlp(pkg, dev, w).forward(x.to(dev))
    assert bool(((y.cpu().double() - want[:, 0]).abs() <= bound[:, 0]).all())


@gpu
@pytest.mark.parametrize("T", [511, 512, 650])
def test_block_shared_expert_of_its_own(pkg, dev, T):
    """An mxfp4 shared expert beside affine experts has launches of its own, over
    every token in order: the block with it less the block without it."""
    E, d, f, K = 16, 256, 192, 4
    nn = pkg.nn
    g = torch.Generator().manual_seed(T)
    w, x, (want, bound) = shared_inputs(T, d, f)
    gate_w = (torch.randn((E, d), generator=g) * 0.1).to(dev)
    sg = (torch.randn((1, d), generator=g) * 0.1).to(dev)
    experts = nn.SplitSwitchFfn.from_dense(*[
        (torch.randn(s, generator=g) * 0.05).bfloat16().to(dev)
        for s in ((E, f, d), (E, f, d), (E, d, f))])
    xd = x.to(dev)
    out = nn.Qwen35MoeBlock(gate_w, experts, K, shared_mlp(pkg, dev, w), sg).forward(xd)
    plain = nn.Qwen35MoeBlock(gate_w, experts, K).forward(xd)
    x64, s64 = x.double(), sg.cpu().double()[0]
    gate = torch.sigmoid(x64 @ s64)[:, None]
    # the gate's logit is an f32 sum of d products, its sigmoid changes by a quarter
    # of that at most and is taken in f32 (a few steps); product and sum round once each
    egate = 0.25 * d * 2.0 ** -23 * (x64.abs() @ s64.abs())[:, None] + 2.0 ** -21
    want, bound = want[:, 0], bound[:, 0]
    big = want.abs() + bound
    tol = gate * bound + egate * big + 2.0 ** -23 * (big + plain.cpu().double().abs())
    diff = out.cpu().double() - plain.cpu().double() - gate * want
    assert bool((diff.abs() <= tol).all())


def test_weights_on_one_device(pkg):
    """A module's tensors on different devices are refused where it is made."""
    nn, Err = pkg.nn, pkg.MlxrMoeError

    def lin(device, rows=64, cols=128, scales=None):
        return nn.QuantizedSwitchLinear(
            torch.zeros((4, rows, cols // 8), dtype=torch.int32, device=device),
            torch.zeros((4, rows, cols // 32), dtype=torch.uint8, device=scales or device),
            mode="mxfp4")

    with pytest.raises(Err, match="different devices"):
        lin("cpu", scales="meta")
    up, down = lin("cpu"), lin("cpu", 128, 64)
    with pytest.raises(Err, match="different devices"):
        nn.SplitSwitchFfn(up, lin("meta"), down)
    with pytest.raises(Err, match="different devices"):
        nn.PackedSwitchFfn(lin("cpu", 128, 128), lin("meta", 128, 64))
    m = nn.SplitSwitchFfn(up, up, down)
    assert m.device == torch.device("cpu")
    with pytest.raises(Err, match="different devices"):
        nn.Qwen35MoeBlock(torch.zeros((4, 128), device="meta"), m, 2)
    with pytest.raises(Err, match="ROCm device"):
        m.forward(torch.zeros((1, 128)).bfloat16(), torch.zeros((1, 2), dtype=torch.int32))


@gpu
def test_weights_on_the_host_are_refused(pkg, dev, tmp_path):
    """Modules made on the host (a checkpoint opened there) take no call."""
    nn, Err = pkg.nn, pkg.MlxrMoeError
    w, x, idx = ffn_inputs(1, 8, 256, 128, 3, 4)
    x, idx = x.to(dev), idx.to(dev)
    m = ffn(pkg, torch.device("cpu"), w)
    wts = torch.ones((3, 4), device=dev)
    gu = [torch.cat([w[0][i], w[1][i]], 1) for i in (0, 1)]
    packed = nn.PackedSwitchFfn(nn.QuantizedSwitchLinear(*gu, mode="mxfp4"), m.down_proj)
    for mod in (m, packed):
        for call in (lambda: mod.forward(x, idx), lambda: mod.forward_with_combine(x, idx, wts)):
            with pytest.raises(Err, match="weights on cpu"):
                call()
    one = [nn.QuantizedLinear(q[0], s[0], mode="mxfp4") for q, s in w]
    with pytest.raises(Err, match="weights on cpu"):
        nn.SwigluMlp(*one).forward(x)
    with pytest.raises(Err, match="ROCm device"):
        one[0].forward(x)
    write_checkpoint(tmp_path)
    block = pkg.loader.qwen35_moe_block(tmp_path, 2, "cpu")
    with pytest.raises(Err, match="weights on cpu"):
        block.forward(x)
    with pytest.raises(Err, match="weights on cpu"):
        block.forward_residual(x, nn.RmsNorm(torch.ones(256, device=dev)))


@gpu
@pytest.mark.parametrize("mode", ["affine", "mxfp4"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T", [1, 3, 40, 300, 600, 7000])
def test_rows_left_out_are_zero(pkg, dev, T, packed, mode):
    """Choices that name no expert, -1 or out of range: their rows of the expert
    outputs are zeros and the weighted sum goes without them, whatever outputs and
    workspace held before; from one token to more rows than the tiles' sort takes."""
    E, d, f, K = 8, 256, 128, 4
    C, lib = pkg._capi, pkg._capi.lib()
    g = torch.Generator().manual_seed(T)
    w = [(torch.randn(s, generator=g) * 0.05).bfloat16().to(dev)
         for s in ((E, f, d), (E, f, d), (E, d, f))]
    if packed:
        m = pkg.nn.PackedSwitchFfn.from_dense(torch.cat(w[:2], 1), w[2], mode=mode)
        experts, forward = lib.mlxr_moe_packed_switch_glu_experts, \
            lib.mlxr_moe_packed_switch_glu_forward
    else:
        m = pkg.nn.SplitSwitchFfn.from_dense(*w, mode=mode)
        experts, forward = lib.mlxr_moe_switch_glu_experts, lib.mlxr_moe_switch_glu_forward
    x = torch.randn((T, d), generator=g).bfloat16().to(dev)
    full = torch.randint(0, E, (T, K), generator=g, dtype=torch.int32)
    out_of = torch.rand((T, K), generator=g) < 0.3
    out_of[0, 1], out_of[0, 0] = True, False
    out_of[T // 2 + 1:T // 2 + 20] = True  # tokens without any expert
    wts = torch.randn((T, K), generator=g).to(dev)
    want = m.forward(x, full.to(dev))
    n = lib.mlxr_moe_packed_switch_glu_workspace_size if packed else \
        lib.mlxr_moe_switch_glu_workspace_size
    ws = torch.empty(n(ctypes.byref(m.descriptor()), T, K), dtype=torch.uint8, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    for value, status in ((-1, 0), (E + 3, 1), (-7, 1)):
        idx = torch.where(out_of, value, full).to(dev)
        y = torch.full((T, K, d), float("nan"), dtype=torch.bfloat16, device=dev)
        ws.fill_(255)
        C.check(experts(ctypes.byref(m.descriptor()), x.data_ptr(), T, idx.data_ptr(), K,
                        y.data_ptr(), ws.data_ptr(), ws.numel(), stream))
        assert pkg.ops.workspace_status(ws) == status
        assert bool((y[out_of] == 0).all())
        # (the kernels may group the rows that are left in another form: an f32 sum and a
        # bf16 step of it)
        keep = ~out_of
        gap = (y[keep].double() - want[keep].double()).abs()
        assert float(gap.norm()) <= 2.0 ** -7 * float(want[keep].double().norm())
        out = torch.full((T, d), float("nan"), device=dev)
        ws.fill_(255)
        kind = (C.FLOAT32,) if packed else ()
        C.check(forward(ctypes.byref(m.descriptor()), x.data_ptr(), T, idx.data_ptr(),
                        wts.data_ptr(), *kind, K, out.data_ptr(), ws.data_ptr(), ws.numel(),
                        stream))
        terms = y.double() * wts.double()[:, :, None]
        assert bool(((out.double() - terms.sum(1)).abs()
                     <= 2 * K * 2.0 ** -24 * terms.abs().sum(1)).all())


@gpu
@pytest.mark.parametrize("T", [3, 40, 300])
def test_outputs_at_any_address(pkg, dev, T):
    """Expert outputs at an address the tiles do not take (two bytes past an
    aligned one): the streaming kernel runs, and rows left out are cleared too."""
    E, d, f, K = 8, 256, 128, 4
    C, lib = pkg._capi, pkg._capi.lib()
    w, x, idx = ffn_inputs(T, E, d, f, T, K)
    want, bound = glu64(x.double(), [values64(*b) for b in w], idx, "swiglu")
    m, xd = ffn(pkg, dev, w), x.to(dev)
    cut = torch.zeros((T, K), dtype=torch.bool)
    cut[T // 2, 1] = cut[T - 1] = True
    store = torch.full((1 + T * K * d,), float("nan"), dtype=torch.bfloat16, device=dev)
    ws = torch.empty(m.workspace_size(T, K), dtype=torch.uint8, device=dev)
    ids = torch.where(cut, -1, idx).to(dev)
    C.check(lib.mlxr_moe_switch_glu_experts(
        ctypes.byref(m.descriptor()), xd.data_ptr(), T, ids.data_ptr(), K, store[1:].data_ptr(),
        ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    y = store[1:].view(T, K, d).cpu().double()
    assert bool(torch.isnan(store[0])) and bool((y[cut] == 0).all())
    assert bool(((y - want).abs() <= bound)[~cut].all())


@gpu
def test_calls_make_their_device_the_current_one(pkg, dev, monkeypatch):
    """Every call launches with its arrays' device current, whichever was before."""
    ops, nn = pkg.ops, pkg.nn
    real, seen = ops._on, []

    def on(t):
        seen.append(t.device)
        return real(t)

    monkeypatch.setattr(ops, "_on", on)
    g = torch.Generator().manual_seed(0)
    x = torch.randn((4, 128), generator=g).bfloat16().to(dev)
    gate = torch.randn((8, 128), generator=g).to(dev)
    w = [torch.randn(s, generator=g).bfloat16().to(dev) * 0.1
         for s in ((8, 64, 128), (8, 64, 128), (8, 128, 64))]
    idx, wts, z = ops.router_topk(x, gate, 2, return_logits=True)
    bf = nn.Linear(gate.bfloat16())
    norm = nn.RmsNorm(torch.ones(128, device=dev))
    for mode in ("affine", "mxfp4"):
        wq, sc, bi = ops.quantize(w[0], mode=mode)
        split = nn.SplitSwitchFfn.from_dense(*w, mode=mode)
        packed = nn.PackedSwitchFfn.from_dense(torch.cat(w[:2], 1), w[2], mode=mode)
        block = nn.Qwen35MoeBlock(gate, split, 2)
        y = split.forward(x, idx)
        _, counts, _, tokens = ops.router_balance(z, idx)
        router = nn.GemmaRouter(gate, torch.ones(128, device=dev), torch.ones(8, device=dev), 2)
        calls = [
            lambda: ops.quantize(w[0], mode=mode),
            lambda: ops.dequantize(wq, sc, bi, mode=mode),
            lambda: ops.gather_qmm(x[:, None, None], wq, sc, bi, rhs_indices=idx, mode=mode),
            lambda: ops.gather_mm(x[:, None, None], w[0], rhs_indices=idx),
            lambda: ops.argpartition_axis(gate, 2, -1), lambda: ops.softmax_axis(gate, -1),
            lambda: ops.router_topk(x, gate, 2), lambda: ops.router_topk_quantized(x, bf, 2),
            lambda: ops.dispatch(idx.reshape(-1), 8), lambda: ops.combine(y, wts),
            lambda: ops.router_balance(z, idx),
            lambda: ops.router_balance_vjp(z, idx, counts, tokens, dweights=wts),
            lambda: ops.workspace_status(split.last_workspace),
            lambda: split.forward(x, idx), lambda: split.forward_with_combine(x, idx, wts),
            lambda: packed.forward(x, idx), lambda: packed.forward_with_combine(x, idx, wts),
            lambda: block.forward(x), lambda: block.forward_residual(x, norm),
            lambda: norm.forward(x), lambda: router.forward(x),
            lambda: nn.GemmaMoe(router, packed).forward(x),
        ]
        for i, call in enumerate(calls):
            seen.clear()
            call()
            assert seen and all(d == x.device for d in seen), i


@gpu
@pytest.mark.parametrize("mode", ["affine", "mxfp4"])
@pytest.mark.parametrize("E,N,K", [(6, 64, 128), (12, 512, 1024)])
def test_strided_weights(pkg, dev, mode, E, N, K):
    """Weights, scales and biases that are views in another order, all at once: the
    copies a call makes of them live until it is done."""
    ops = pkg.ops
    g = torch.Generator(device=dev).manual_seed(K)
    w = torch.randn((E, N, K), generator=g, device=dev).bfloat16()
    parts = ops.quantize(w, mode=mode)
    x = torch.randn((5, 1, K), generator=g, device=dev).bfloat16()
    idx = torch.arange(5, dtype=torch.int32, device=dev)

    def turned(t):  # the same values, rows not one after another
        return None if t is None else t.transpose(0, 1).contiguous().transpose(0, 1)

    for _ in range(3):
        views = [turned(t) for t in parts]
        torch.cuda.synchronize()
        assert torch.equal(ops.dequantize(*views, mode=mode), ops.dequantize(*parts, mode=mode))
        a = ops.gather_qmm(x, *views, rhs_indices=idx, mode=mode)
        assert torch.equal(a, ops.gather_qmm(x, *parts, rhs_indices=idx, mode=mode))
    y = torch.randn((40, 4, K), generator=g, device=dev).bfloat16()
    wts = torch.rand((40, 4), generator=g, device=dev)
    sy = torch.randn((40, K), generator=g, device=dev).bfloat16()
    z = torch.randn((40,), generator=g, device=dev)
    flat = [t.t().contiguous().t() for t in (wts, sy)]
    wide = torch.stack([z, z], 1)[:, 0]
    assert torch.equal(ops.combine(turned(y), flat[0], flat[1], wide), ops.combine(y, wts, sy, z))


def test_combine_takes_a_weight_per_choice(pkg):
    nn, Err = pkg.nn, pkg.MlxrMoeError

    def lin(rows, cols):
        return nn.QuantizedSwitchLinear(torch.zeros((4, rows, cols // 8), dtype=torch.int32),
                                        torch.zeros((4, rows, cols // 32), dtype=torch.uint8),
                                        mode="mxfp4")

    split = nn.SplitSwitchFfn(lin(64, 128), lin(64, 128), lin(128, 64))
    packed = nn.PackedSwitchFfn(lin(128, 128), lin(128, 64))
    x, idx = torch.zeros((6, 128)).bfloat16(), torch.zeros((6, 2), dtype=torch.int32)
    for m in (split, packed):
        for bad in (torch.ones(5, 2), torch.ones(6, 1), torch.ones(4, 3), torch.ones(6)):
            with pytest.raises(Err, match="must match indices"):
                m.forward_with_combine(x, idx, bad)
        with pytest.raises(Err, match="ROCm device"):
            m.forward_with_combine(x, idx, torch.ones(6, 2))
