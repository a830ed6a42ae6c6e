"""Sums of e4m3 products where large ones cancel: within the stated bound with a bf16 output, exact to FP32 with an f32 one.

Bounds per element: with a bf16 output k 2^-13 of the largest |x w| of the sum (what the 8-bit matrix instruction may drop),
k 2^-23 of the magnitudes' sum and half a rounding; with an f32 output k 2^-23 of the magnitudes' sum (each of k additions
rounds once, the scales and the output once more)."""
import math

import pytest

torch = pytest.importorskip("torch")

from julia1_amd import hip  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn

# (rows, n, k) of a kernel each: up to 16 rows, 64 x 64 tiles, 128 x 128 one and two to a CU, 128 x 256, 256 x 256
SIZES = {"stream": (5, 72, 1040), "small": (40, 72, 1040), "deep": (1000, 4000, 528), "pair": (1500, 4000, 528),
         "tall": (1100, 4000, 1040), "wide": (3900, 4000, 528)}


def operands(rows, n, k):
    """Small codes everywhere; per row two strong channels whose products cancel in every even column, and per every
    third column one that stands alone."""
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = (torch.randn(rows, k, device="cuda", generator=g) / 2).to(E4M3).float()
    w = (torch.randn(n, k, device="cuda", generator=g) / 4).to(E4M3).float()
    for a, b in ((3, 9), (k - 6, k - 1)):
        x[:, a] = x[:, b] = 256.0
        w[:, a], w[:, b] = 192.0, -192.0
        w[1::2, b] = 96.0
    w[::3, 20] = 448.0
    xs, ws = (0.5 + torch.rand(c, device="cuda", generator=g) for c in (rows, n))
    return x.to(E4M3), w.to(E4M3), xs, ws


def some(rows):
    return torch.arange(rows, device="cuda") if rows < 100 else torch.tensor([0, 17, rows // 2, rows - 1], device="cuda")


def bounds(x, w, xs, ws, i):
    """z of rows i, the largest product, the sum of magnitudes, in 64 bits."""
    xd, wd = x[i].double() * xs[i].double()[:, None], w.double() * ws.double()[:, None]
    top = torch.stack([(r.abs() * wd.abs()).amax(dim=1) for r in xd])
    return xd @ wd.t(), top, xd.abs() @ wd.abs().t()


@pytest.mark.parametrize("kernel", list(SIZES))
def test_cancelling_products(kernel):
    rows, n, k = SIZES[kernel]
    assert hip.linear_plan("linear", E4M3, rows, n, k) == [(kernel, 1, rows)]
    x, w, xs, ws = operands(rows, n, k)
    half, full = torch.empty(rows, n, device="cuda", dtype=BF16), torch.empty(rows, n, device="cuda")
    hip.op_linear(x, w, half, x_scale=xs, w_scale=ws)
    hip.op_linear(x, w, full, x_scale=xs, w_scale=ws)
    torch.cuda.synchronize()
    i = some(rows)
    z, top, size = bounds(x, w, xs, ws, i)
    off = (half[i].double() - z).abs() - k * 2.0**-13 * top - size * (k + 4) * 2.0**-23
    assert float((off - (z.abs() + k * 2.0**-13 * top) * 2.0**-8).max()) <= 0
    assert float(((full[i].double() - z).abs() - size * (k + 4) * 2.0**-23).max()) <= 0
    # what the f32 output keeps where the strong products cancel: the small ones, well above its own error
    rest = z[:, ::2].abs().median()
    assert float(((full[i] - z)[:, ::2]).abs().max()) < float(rest) / 4


@pytest.mark.parametrize("rows,n,k", [(5, 72, 1040), (40, 72, 1040), (1100, 2000, 1040), (1500, 2000, 528), (3900, 2000, 528)])
def test_cancelling_products_gated(rows, n, k):
    x, w, xs, ws = operands(rows, 2 * n, k)
    w[n:] = 0
    w[n:, 1] = 1.0
    x[:, 1] = 1.0
    xs.fill_(1.0)
    ws.fill_(1.0)
    out = torch.empty(rows, n, device="cuda", dtype=BF16)
    hip.op_gated_ffn(x, w, out, act="none", x_scale=xs, w_scale=ws)  # the gate's sums, times 1
    torch.cuda.synchronize()
    i = some(rows)
    z, top, size = bounds(x, w[:n], xs, ws[:n], i)
    off = (out[i].double() - z).abs() - k * 2.0**-13 * top - size * (k + 4) * 2.0**-23
    assert float((off - (z.abs() + k * 2.0**-13 * top) * 2.0**-8).max()) <= 0
