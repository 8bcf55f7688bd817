"""The large tiles of the products over sorted rows -- what long prompts and training passes
take -- over ragged groups, every row against a plain 64-bit form.

Tolerances as in test_grouped.py."""
import pytest
import torch

from test_grouped import BF16, F32, forward64, near, problem, taken, to

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
