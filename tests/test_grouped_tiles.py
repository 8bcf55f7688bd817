"""The large tiles of the products over sorted rows -- what long prompts and training passes
take -- over ragged groups, every row against a plain 64-bit form; and how exact the products of
8- by 4-bit codes are.

Tolerances of the bf16 products as in test_grouped.py.  The matrix instructions of the codes
add eight neighbouring products at a time; they cut each toward zero at 2^-13 of the largest
one's power of two, the sum of its factors' exponents as the codes hold them (a product of zero
has none, and a code below the smallest normal one the exponent of that).  `cut_products` does
the same in 64 bits.  What is left is a sum of K terms in f32: off by at most K * 2^-24 of the
sum of their magnitudes."""
import pytest
import torch

from test_add_norm import decode8
from test_grouped import BF16, F32, forward64, near, problem, taken, to, values4

gpu = pytest.mark.gpu

COUNTS = [1, 33, 129, 255, 0, 300, 600, 128, 257, 64]


def ceil(a, b):
    return (a + b - 1) // b


def parts(R, E, rows):
    return R // rows + min(R, E + 2)


def forward_kernel(R, E, N, K, codes=False):
    """Which kernel a product takes."""
    few = parts(R, E, 64) * ceil(N, 128) < 256
    if R <= (8 * E if few else 4 * E * (K <= 512) if codes else 2 * E):
        return "stream"
    cols, rows_most = (128, 32 * E) if codes else (256, 64 * E)
    if R <= rows_most or parts(R, E, 128) * ceil(N, cols) < 256:
        return "64 x 128"
    return f"128 x {cols}"


def dx_kernel(R, E, N, K):
    return "64 x 128" if parts(R, E, 128) * ceil(K, 256) < 256 else "128 x 256"


def loose_rows(rows, mapped):
    """A ninth of the indices name no row."""
    if rows is not None:
        rows[4::9] = torch.tensor([-1, mapped, 2 ** 31 - 1], dtype=torch.int32).repeat(
            rows.numel())[: rows[4::9].numel()]
    return rows


@gpu
@pytest.mark.parametrize("K,N", [(72, 2824), (264, 3000), (2824, 72), (3000, 136)])
@pytest.mark.parametrize("mapped", [None, 400])
def test_large_tiles(pkg, dev, K, N, mapped):
    """The forward product (N wide), dx (K wide) and dW of ten groups."""
    R, E = sum(COUNTS) + 7, len(COUNTS)
    wide = forward_kernel(R, E, N, K), dx_kernel(R, E, N, K)
    assert wide == (("128 x 256", "64 x 128") if N > K else ("64 x 128", "128 x 256"))
    x, w, dy, offsets, rows = problem(K - N + 9999, COUNTS, K, N, tail=7, mapped=mapped)
    rows = loose_rows(rows, mapped)
    xs = taken(x, rows)
    y, mass = forward64(xs, w, offsets)
    for out_dtype in (BF16, F32):
        got = pkg.ops.grouped_mm(*to(dev, x, w, offsets, rows), out_dtype=out_dtype)
        near(got, y, mass, K)
        assert bool((got[-7:] == 0).all())
    dx, dw = pkg.ops.grouped_mm_vjp(*to(dev, dy, x, w, offsets, rows), dw_dtype=F32)
    g = dy.double()
    near(dx, *forward64(g, w.transpose(1, 2), offsets), N)
    assert bool((dx[-7:] == 0).all())
    for e in range(E):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        ok = xs[s].abs().sum(1) > 0 if mapped else torch.ones(s.stop - s.start, dtype=torch.bool)
        near(dw[e], g[s][ok].t() @ xs[s][ok], g[s][ok].abs().t() @ xs[s][ok].abs(), COUNTS[e] + 1)


def exponents8(q, sc):
    """The exponent of each e4m3 code under its scale, as the code holds it."""
    b = torch.stack([(q >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2)
    return ((b >> 3) & 15).clamp_min(1) - 7 + sc.long().repeat_interleave(32, -1) - 127


def exponents4(wq, sc):
    """... and of each e2m1 code."""
    b = torch.stack([(wq >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2)
    return ((b >> 1) & 3).clamp_min(1) - 1 + sc.long().repeat_interleave(32, -1) - 127


def cut_products(x, ex, w, ew):
    """(y, mass) of rows x [r, K] by w [N, K] with every eight products cut as said above."""
    y = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    mass = torch.zeros_like(y)
    for k in range(0, x.shape[1], 8):
        p = x[:, None, k:k + 8] * w[None, :, k:k + 8]
        e = ex[:, None, k:k + 8] + ew[None, :, k:k + 8]
        top = torch.where(p != 0, e, -1000).amax(-1, keepdim=True).clamp_min(-900).double()
        unit = torch.exp2(top - 13)
        y += (torch.trunc(p / unit) * unit).sum(-1)
        mass += p.abs().sum(-1)
    return y, mass


# counts, K, N and the kernel that takes them: whole and odd K (scales by words and by bytes)
CODES = [([1, 0, 3, 2] + [0] * 20, 160, 40, "stream"),
         ([1, 0, 3, 2] + [0] * 20, 2176, 24, "stream"),
         ([3, 40, 0, 100, 64], 160, 264, "64 x 128"),
         ([3, 40, 0, 100, 64], 1024, 72, "64 x 128"),
         ([1, 33, 129, 255, 0, 300, 600], 160, 2040, "128 x 128"),
         ([1, 33, 129, 255, 0, 300, 600], 640, 2048, "128 x 128")]


@gpu
@pytest.mark.parametrize("counts,K,N,kernel", CODES)
@pytest.mark.parametrize("mapped", [None, 130])
@pytest.mark.parametrize("spread", [0, 9])
def test_products_of_codes(pkg, dev, counts, K, N, kernel, mapped, spread):
    """f32 outputs, and bf16 ones as those rounded; values alike and 2^spread apart."""
    E, R = len(counts), sum(counts) + 5
    assert forward_kernel(R, E, N, K, True) == kernel
    x, w, _, offsets, rows = problem(K + N + spread, counts, K, N, tail=5, mapped=mapped)
    rows = loose_rows(rows, mapped)
    g = torch.Generator().manual_seed(K)

    def apart(shape):
        return torch.exp2(torch.randint(-spread, spread + 1, shape, generator=g).float())

    x = x.float() * apart(x.shape) * apart((x.shape[0], K // 32)).repeat_interleave(32, -1)
    q, sc, _ = pkg.ops.quantize(x.to(dev), mode="mxfp8")
    wq, wsc, _ = pkg.ops.quantize(w.to(dev), mode="mxfp4")
    od, rd = to(dev, offsets, rows)
    got = pkg.ops.grouped_qmm(q, sc, wq, wsc, od, rd, out_dtype=F32)
    half = pkg.ops.grouped_qmm(q, sc, wq, wsc, od, rd)
    assert torch.equal(half, got.to(BF16)) and bool((got[-5:] == 0).all())
    src = torch.arange(R) if rows is None else rows
    named = (src >= 0) & (src < x.shape[0])
    src = torch.where(named, src, 0).long().to(dev)
    assert bool((got[~named.to(dev)] == 0).all())
    xv, wv = decode8(q.cpu(), sc.cpu()).to(dev), values4(wq.cpu(), wsc.cpu()).to(dev)
    ex, ew = exponents8(q, sc), exponents4(wq, wsc)
    for e in range(E):
        r = torch.arange(int(offsets[e]), int(offsets[e + 1]))
        r = r[named[r]].to(dev)
        if not len(r):
            continue
        y, mass = cut_products(xv[src[r]], ex[src[r]], wv[e], ew[e])
        err = (got[r].double() - y).abs()
        assert bool((err <= K * 2.0 ** -24 * mass + 1e-38).all()), float((err / mass).max())
