"""Rows at the edge of what the feed-forward operators' contract covers."""
import math

import pytest

torch = pytest.importorskip("torch")

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
