"""Activations of the feed-forward operators where they are small: their relative error, against 64 bits.

Bounds, relative to the value: GELU (8 + z^2) 2^-23 (the cdf's 6 + z^2, a product and a rounding), SiLU (8 + |z|) 2^-23,
the tanh form (8 + 4 |u|) 2^-23 with u the argument of its sigmoid (three roundings, one more and a constant's in the
exponential, those of its own two constants: under 7 of 2^-24 each).  Slopes the same, relative to the sum of their terms'
magnitudes, and for u > 0 another |z u'| 2^-23, as 1 - s is off by 2^-23 of 1.  Values whose sigmoid or exponential is
below 2^-126 may be flushed: up to 2^-119."""
import math

import pytest

torch = pytest.importorskip("torch")

from julia1_amd import hip  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-23
FLUSH = 2.0**-119


def exact(z, act):
    """(value, slope, the bound of either over 2^-23) in 64 bits."""
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, z.abs() * cdf * (8 + z * z), (cdf + z.abs() * pdf) * (8 + z * z)
    a, b = (1.0, 0.0) if act == "silu" else (2 * math.sqrt(2 / math.pi), 0.044715)
    u = a * (z + b * z**3)
    s, t = torch.sigmoid(u), torch.sigmoid(-u)
    du = a * (1 + 3 * b * z * z)
    more, factor = z * s * t * du, 8 + u.abs() * (1 if act == "silu" else 4)
    return z * s, s + more, z.abs() * s * factor, (s + more.abs()) * factor + (z * du).clamp_min(0)


def grid():
    """Values whose bf16 rounding is themselves, to where the results leave FP32's range."""
    z = torch.cat([torch.linspace(-14, 14, 3585), -torch.logspace(-30, 0, 200), torch.logspace(-30, 0, 199),
                   -torch.linspace(14, 87, 512), torch.zeros(8)])
    return z[: z.numel() // 8 * 8].to(BF16).float().cuda()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [1, 40])
def test_small_values(act, rows):
    z = grid()
    n, k = z.numel(), 16
    x, w = torch.zeros(rows, k, device="cuda", dtype=BF16), torch.zeros(n, k, device="cuda", dtype=BF16)
    out = torch.empty(rows, n, device="cuda")
    hip.op_linear(x, w, out, bias=z, act=act)
    # the same of the gated projections, whose other half is 1
    x[:, 0], w[:, 0] = 1, z.to(BF16)
    h = torch.empty(rows, n, device="cuda", dtype=BF16)
    hip.op_gated_ffn(x, torch.cat([w, torch.ones_like(w)]), h, act=act)
    # a row's slope alone is its dbias, in f32
    dy, db = torch.zeros(rows, n, device="cuda", dtype=BF16), torch.empty(n, device="cuda")
    dy[-1] = 1
    ws = torch.empty(hip.linear_backward_workspace(rows, n, k, act), dtype=torch.uint8, device="cuda")
    hip.op_linear_backward(dy, x, w, ws, act=act, pre=w[:, 0].repeat(rows, 1), dbias=db)
    torch.cuda.synchronize()
    value, slope, value_tol, slope_tol = exact(z.double(), act)
    for row in out:
        off = (row.double() - value).abs() - value_tol * U - FLUSH
        assert float(off.max()) <= 0, (act, float(z[off.argmax()]))
    off = (h.double() - value).abs() - value.abs() * 2.0**-8 - value_tol * 1.01 * U - FLUSH
    assert float(off.max()) <= 0, (act, float(z[off.max(dim=0)[0].argmax()]))
    off = (db.double() - slope).abs() - slope_tol * U - FLUSH
    assert float(off.max()) <= 0, (act, float(z[off.argmax()]))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gated_slopes_of_small_values(act):
    """[dg du] of the gated backward, from dwi of one row with x = 1: dh u act'(g), and dh act(g)."""
    z = grid()
    n = z.numel()
    x, dh = torch.zeros(1, 8, device="cuda", dtype=BF16), torch.ones(1, n, device="cuda", dtype=BF16)
    x[:, 0] = 1
    gu, dwi = torch.cat([z.to(BF16), torch.ones_like(z, dtype=BF16)])[None, :], torch.empty(2 * n, 8, device="cuda")
    ws = torch.empty(hip.gated_ffn_backward_workspace(1, n, 8), dtype=torch.uint8, device="cuda")
    hip.op_gated_ffn_backward(dh, gu, x, torch.zeros(2 * n, 8, device="cuda", dtype=BF16), ws, act=act, dw=dwi)
    torch.cuda.synchronize()
    value, slope, value_tol, slope_tol = exact(z.double(), act)
    for got, want, tol in ((dwi[:n, 0], slope, slope_tol), (dwi[n:, 0], value, value_tol)):
        off = (got.double() - want).abs() - want.abs() * 2.0**-8 - tol * 1.01 * U - FLUSH
        assert float(off.max()) <= 0, (act, float(z[off.argmax()]))


@pytest.mark.parametrize("rows", [2, 40])
def test_gelu_of_what_is_not_a_number_or_infinite(rows):
    z = torch.tensor([float("nan"), float("inf"), -1e38, -float("inf"), -0.0, 15.0, -15.0, 1e38], device="cuda")
    x, w = torch.zeros(rows, 16, device="cuda", dtype=BF16), torch.zeros(8, 16, device="cuda", dtype=BF16)
    out = torch.empty(rows, 8, device="cuda")
    hip.op_linear(x, w, out, bias=z, act="gelu")
    torch.cuda.synchronize()
    for row in out.tolist():
        assert math.isnan(row[0]) and row[1] == math.inf and row[2:5] == [0, 0, 0] and row[5] == 15
        assert abs(row[6]) < FLUSH and row[7] == z[7].item()
