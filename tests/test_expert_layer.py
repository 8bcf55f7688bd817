"""The operators of an expert layer together, as a model's step calls them: the residual add
and norm, the router, the sort by expert, the three projections over sorted rows and the
weighted sum; then their gradients back to the layer's input and every weight.

Tolerances: of every result, relative in the root of the sum of squares.  A bf16 rounding is
off by at most 2^-8 of each value, so by 2^-8 in that norm; the products with random weights
pass an error on as they pass the values on, so the roundings on the longest way add up: y,
the SwiGLU, its product and the f32 sum on the way out (3 of 2^-8; counted as 4), and on the
way back 4 more of gradients and the two factors of each weight gradient (counted as 12).  In
mode mxfp8 the rows are taken as the device quantised them, and only bf16 roundings count.
"""
import pytest
import torch
import torch.nn.functional as F

from test_add_norm import decode8
from test_grouped import values4

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-6


def far(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


class Layer:
    """d inputs, E experts of width f, k choices; bf16 weights, the router's in f32."""

    def __init__(self, pkg, dev, seed, d, E, f, k):
        g = torch.Generator().manual_seed(seed)

        def normal(shape, std):
            return torch.randn(shape, generator=g) * std

        self.pkg, self.k, self.E, self.d = pkg, k, E, d
        self.wn = (1 + normal((d,), 0.2)).to(BF16)
        self.wr = normal((E, d), d ** -0.5)
        self.w = [normal(s, s[2] ** -0.5).to(BF16) for s in ((E, f, d), (E, f, d), (E, d, f))]
        nn = pkg.nn
        self.norm = nn.RmsNorm(self.wn.to(dev), EPS)
        self.router = self.wr.to(dev)
        self.gate, self.up, self.down = [nn.SwitchLinear(w.to(dev)) for w in self.w]

    def forward(self, x, residual):
        ops, k, d = self.pkg.ops, self.k, self.d
        h, y = self.norm.forward_add(x, residual)
        idx, wts, logits = ops.router_topk(y, self.router, k, return_logits=True)
        _, offsets, order, inv = ops.dispatch(idx, self.E)
        rows = torch.div(order, k, rounding_mode="floor")
        g = self.gate.apply_grouped(y, offsets, rows, F32)
        u = self.up.apply_grouped(y, offsets, rows, F32)
        a = (F.silu(g) * u).to(BF16)
        o = self.down.apply_grouped(a, offsets)
        out = ops.combine(o[inv.long()].view(-1, k, d), wts)
        return out, (h, y, idx, wts, logits, offsets, order, inv, rows, g, u, a, o)

    def backward(self, dout, dh, kept):
        """Gradients of <dout, out> + <dh, h>: of x, the norm's, the router's and the experts'
        weights."""
        ops, k, d = self.pkg.ops, self.k, self.d
        h, y, idx, wts, logits, offsets, order, inv, rows, g, u, a, o = kept
        sorted_w = wts.reshape(-1)[order.long()]
        taken = dout[rows.long()]
        do = (taken * sorted_w[:, None]).to(BF16)
        da, dwd = self.down.vjp_grouped(do, a, offsets, dw_dtype=F32)
        s = torch.sigmoid(g)
        da = da.float()
        du = (da * g * s).to(BF16)
        dg = (da * u * s * (1 + g * (1 - s))).to(BF16)
        dxg, dwg = self.gate.vjp_grouped(dg, y, offsets, rows, dw_dtype=F32)
        dxu, dwu = self.up.vjp_grouped(du, y, offsets, rows, dw_dtype=F32)
        one = torch.ones_like(wts)
        back = inv.long()
        dy = (ops.combine(dxg[back].view(-1, k, d), one)
              + ops.combine(dxu[back].view(-1, k, d), one))
        dweights = (taken * o.float()).sum(-1)[back].view(wts.shape)
        dlogits = ops.router_balance_vjp(logits, idx, dweights=dweights)
        dy = dy + dlogits @ self.router
        dx, dwn = self.norm.vjp(dy, h, dh)
        return dx, dwn, dlogits.t() @ y.float(), dwg, dwu, dwd


def plain(layer, x, residual, idx, dout, dh):
    """The same in 64 bits, by differentiation, with the routing given."""
    x, residual = x.double(), residual.double()
    x.requires_grad_()
    par = [t.double().requires_grad_() for t in (layer.wn, layer.wr, *layer.w)]
    wn, wr, wg, wu, wd = par
    h = x + residual
    y = wn * h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    p = torch.softmax(y @ wr.t(), -1).gather(1, idx.long())
    wts = p / p.sum(-1, keepdim=True)
    out = torch.zeros_like(y)
    for t in range(y.shape[0]):
        e = idx[t].long()
        a = F.silu(wg[e] @ y[t]) * (wu[e] @ y[t])
        out[t] = (wts[t][:, None] * torch.einsum("kdf,kf->kd", wd[e], a)).sum(0)
    loss = (out * dout.double()).sum() + (h * dh.double()).sum()
    return out.detach(), torch.autograd.grad(loss, [x] + par)


@gpu
@pytest.mark.parametrize("T,d,E,f,k,stream", [(1, 64, 4, 32, 2, BF16), (70, 136, 16, 72, 3, BF16),
                                              (333, 64, 5, 200, 2, F32), (40, 256, 200, 64, 8, F32)])
def test_layer_and_its_gradients(pkg, dev, T, d, E, f, k, stream):
    layer = Layer(pkg, dev, T, d, E, f, k)
    g = torch.Generator().manual_seed(d)
    x = torch.randn((T, d), generator=g)
    residual = torch.randn((T, d), generator=g).to(stream)
    # (h as the stream keeps it, so that both norms are of the same values)
    residual = ((x + residual.float()).to(stream).double() - x.double()).to(F32)
    dout, dh = torch.randn((T, d), generator=g), torch.randn((T, d), generator=g).to(stream)
    if stream == BF16:
        x = torch.zeros_like(x)
        residual = residual.to(BF16)
    out, kept = layer.forward(x.to(dev), residual.to(dev))
    grads = layer.backward(dout.to(dev), dh.to(dev), kept)
    want, dwant = plain(layer, x, residual, kept[2].cpu(), dout, dh)
    assert far(out, want) <= 4 * 2.0 ** -8
    for name, a, b in zip(("x", "norm", "router", "gate", "up", "down"), grads, dwant):
        assert far(a, b) <= 12 * 2.0 ** -8, name


@gpu
def test_layer_in_a_graph(pkg, dev):
    """A whole step captured, and replayed with other inputs and so another routing."""
    layer = Layer(pkg, dev, 5, 128, 12, 64, 2)
    x, residual = torch.randn((50, 128), device=dev), torch.randn((50, 128), device=dev)
    dout, dh = torch.randn_like(x), torch.randn_like(x)

    def step():
        out, kept = layer.forward(x, residual)
        return (out, kept[2], *layer.backward(dout, dh, kept))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            got.append(step())
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        for t in (x, residual, dout, dh):
            t.copy_(torch.randn(t.shape, generator=g))
        for graph in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
@pytest.mark.parametrize("T,d,E,f,k", [(1, 64, 8, 32, 2), (5, 256, 16, 96, 4),
                                       (300, 128, 6, 160, 2)])
def test_microscaled_layer(pkg, dev, T, d, E, f, k):
    """Rows normed to mxfp8, experts in mxfp4: the gate, up and down projections."""
    ops, nn = pkg.ops, pkg.nn
    layer = Layer(pkg, dev, d + T, d, E, f, k)
    gate, up, down = [l.try_into_quantized(mode="mxfp4")
                      for l in (layer.gate, layer.up, layer.down)]
    g = torch.Generator().manual_seed(f)
    x, residual = torch.randn((T, d), generator=g), torch.randn((T, d), generator=g).to(BF16)
    idx = torch.rand((T, E), generator=g).topk(k, 1).indices.int()
    wts = torch.rand((T, k), generator=g)
    _, q, sc = layer.norm.forward_add(x.to(dev), residual.to(dev), mode="mxfp8")
    _, offsets, order, inv = ops.dispatch(idx.to(dev), E)
    rows = torch.div(order, k, rounding_mode="floor")
    a = F.silu(gate.apply_grouped(q, sc, offsets, rows, F32))
    a = a * up.apply_grouped(q, sc, offsets, rows, F32)
    aq, asc, _ = ops.quantize(a, mode="mxfp8")
    o = down.apply_grouped(aq, asc, offsets)
    out = ops.combine(o[inv.long()].view(T, k, d), wts.to(dev))

    wg, wu, wd = [values4(l.weight.cpu(), l.scales.cpu()) for l in (gate, up, down)]
    y = decode8(q.cpu(), sc.cpu())
    act = decode8(aq.cpu(), asc.cpu())
    want_a, want = torch.zeros((T * k, f), dtype=torch.float64), torch.zeros((T, d)).double()
    for i, (t, c) in enumerate((int(v) // k, int(v) % k) for v in order.cpu()):
        e = int(idx[t, c])
        want_a[i] = F.silu(wg[e] @ y[t]) * (wu[e] @ y[t])
        want[t] += wts[t, c].double() * (wd[e] @ act[i])
    assert far(a, want_a) <= 2.0 ** -8  # (f32: only what the matrix instructions drop)
    assert far(out, want) <= 2 * 2.0 ** -8
    with pytest.raises(pkg.MlxrMoeError, match="mode mxfp4"):
        nn.QuantizedSwitchLinear.try_from_switch_linear(layer.gate.weight, 32).apply_grouped(
            q, sc, offsets, rows)
