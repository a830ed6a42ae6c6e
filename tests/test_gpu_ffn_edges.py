"""Rows at the edge of what the feed-forward operators' contract covers."""
import math

import pytest

torch = pytest.importorskip("torch")

from ffn_routes import ROUTES  # noqa: E402
from julia1_amd import hip  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.mark.parametrize("h", [8, 768, 5000])
@pytest.mark.parametrize("xt", [BF16, F16, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_rows_of_zeros_and_of_nothing_but_nan_in_eight_bits(h, xt, eps):
    """A row of zeros, or one that w makes zeros, has codes and scale 0 whatever eps; a NaN's row keeps its NaN."""
    x = torch.zeros(4, h, device="cuda", dtype=xt)
    x[1, 0] = 3.0
    x[2] = float("nan")
    x[3, 1] = -2.0
    w = torch.ones(h, device="cuda")
    w[1] = 0.0
    out, scales = torch.full((4, h), 1.0, device="cuda").to(E4M3), torch.full((4,), 7.0, device="cuda")
    hip.op_rms_norm(x, w, eps, out, scales=scales)
    torch.cuda.synchronize()
    for r in (0, 3):
        assert scales[r].item() == 0 and not bool(out[r].float().any())
    assert out[1, 0].float().item() == 448 and not bool(out[1, 1:].float().any())
    want = 3.0 / math.sqrt(9.0 / h + eps) / 448
    assert abs(scales[1].item() / want - 1) < 2.0**-20
    assert bool(out[2].float().isnan().all()) and math.isnan(scales[2].item())


@pytest.mark.parametrize("out_t", [BF16, F32])
@pytest.mark.parametrize("name", ["stream", "small", "deep", "pair", "tall", "wide"])
def test_e4m3_not_a_number_stays_in_its_row_and_column(name, out_t):
    """A NaN code of x spoils its output row, one of w its output column, and nothing else."""
    rows, n, k = ROUTES["linear", "e4m3"][name]
    x, w = torch.ones(rows, k, device="cuda").to(E4M3), torch.ones(n, k, device="cuda").to(E4M3)
    x[rows // 2, k - 1] = float("nan")
    w[n - 3, 0] = float("nan")
    out = torch.zeros(rows, n, device="cuda", dtype=out_t)
    hip.op_linear(x, w, out)
    torch.cuda.synchronize()
    want = torch.full((rows, n), float(k), device="cuda").to(out_t)
    want[rows // 2], want[:, n - 3] = float("nan"), float("nan")
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("name", ["small", "small/parts", "deep", "deep/parts", "pair", "pair/parts", "wide", "wide/parts"])
def test_gradients_of_not_a_number_stay_in_their_row_and_column(name):
    """A NaN of dy spoils its row of dx and its row of dw (an output feature's), one of w its column of dx, one of x its
    column of dw, and nothing else: not through the zeros that stand for what lies past an end."""
    for product in ("dx", "dw"):
        rows, n, k = ROUTES[product, "half"][name]
        dy, x, w = (torch.ones(*s, device="cuda", dtype=BF16) for s in ((rows, n), (rows, k), (n, k)))
        dy[rows // 2, n - 3] = w[n - 1, 5] = x[rows - 1, k - 2] = float("nan")
        dx, dw = torch.zeros(rows, k, device="cuda", dtype=BF16), torch.zeros(n, k, device="cuda")
        ws = torch.empty(hip.linear_backward_workspace(rows, n, k), dtype=torch.uint8, device="cuda")
        hip.op_linear_backward(dy, x, w, ws, **({"dx": dx} if product == "dx" else {"dw": dw}))
        torch.cuda.synchronize()
        if product == "dx":
            got, want = dx, torch.full((rows, k), float(n), device="cuda").to(BF16)
            want[rows // 2], want[:, 5] = float("nan"), float("nan")
        else:
            got, want = dw, torch.full((n, k), float(rows), device="cuda")
            want[n - 3], want[:, k - 2] = float("nan"), float("nan")
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num()), product


@pytest.mark.parametrize("name", ["stream", "small", "deep", "pair", "tall", "wide", "wide+small", "wide+pair"])
def test_residual_in_place_on_every_kernel(name):
    """resid may be out, where a product takes two launches too."""
    rows, n, k = ROUTES["linear", "half"][name]
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w = (torch.randn(*s, device="cuda", generator=g).to(BF16) for s in ((rows, k), (n, k)))
    for out_t in (BF16, F32):
        resid = torch.randn(rows, n, device="cuda", generator=g).to(out_t)
        apart = torch.empty_like(resid)
        hip.op_linear(x, w, apart, resid=resid, act="gelu")
        hip.op_linear(x, w, resid, resid=resid, act="gelu")
        torch.cuda.synchronize()
        assert torch.equal(apart, resid)
