"""The kernels that products are put on by their sizes, asked from the library: no device is needed."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from ffn_routes import ROUTES, route  # noqa: E402
from julia1_amd import abi, hip  # noqa: E402

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
# columns and rows of a tile, threads
TILE = {"small": (64, 64, 256), "deep": (128, 128, 512), "pair": (128, 128, 256),
        "tall": (128, 256, 512), "wide": (256, 256, 512)}


def threads(product, launch, cols):
    """Threads along x of one launch."""
    kernel, _, rows = launch
    if kernel == "stream":
        return -(-cols // 16) * 512
    p, q, t = TILE[kernel]
    return -(-cols * (2 if product == "gated" else 1) // p) * -(-rows // q) * t


def check_launchable(product, dtype, rows, n, k, out=None):
    launches = hip.linear_plan(product, dtype, rows, n, k, out)
    cols = k if product in ("dx", "dw") else n
    assert sum(r for _, _, r in launches) == (n if product == "dw" else rows)
    for launch in launches:
        assert threads(product, launch, cols) < 1 << 32, launch
    return launches


# both sides of where 64 x 64 tiles of 256 threads (2^24 of them), and tiles of 512 threads (2^23), pass 2^32 threads
@pytest.mark.parametrize("rows", [(1 << 30) - 64, (1 << 30) - 63, 1 << 30, (1 << 29) + 1, 1 << 29, 1 << 28, (1 << 27) + 5])
@pytest.mark.parametrize("dtype,out", [(BF16, None), (F16, F32), (E4M3, None), (E4M3, F32)])
def test_products_of_many_rows_have_a_launch(rows, dtype, out):
    """As many rows as the header promises, with as many columns as the card's memory holds."""
    for n, k in ((8, 16), (8, 64), (64, 16), (120, 16)):
        check_launchable("linear", dtype, rows, n, k, out)
        if out is None:
            check_launchable("gated", dtype, rows, n, k)


@pytest.mark.parametrize("rows", [(1 << 30) - 63, 1 << 30, 1 << 29])
def test_gradients_of_many_rows_have_a_launch(rows):
    for n, k in ((8, 8), (16, 64), (128, 16)):
        check_launchable("dx", BF16, rows, n, k)
        check_launchable("dw", BF16, rows, n, k)


def test_small_tiles_up_to_what_a_launch_holds():
    """The last size on 64 x 64 tiles and the first past them."""
    assert hip.linear_plan("linear", BF16, (1 << 30) - 64, 8, 8) == [("small", 1, (1 << 30) - 64)]
    (kernel, _, _), = hip.linear_plan("linear", BF16, 1 << 30, 8, 8)
    assert kernel != "small"


def test_gradients_that_no_launch_holds_are_refused_at_once():
    """Before anything is launched (a device is not needed for the refusal), and by the workspace's size too."""
    rows, n, k, a = 1 << 30, 16, 1 << 18, 1 << 52  # addresses are made up and far apart
    for act, pre in ((abi.ACT_NONE, None), (abi.ACT_GELU, a)):
        assert hip.lib().jh_op_linear_backward(abi.BF16, 2 * a, n, 3 * a, k, rows, 4 * a, n, k, act, pre, n, 5 * a, k,
                                               abi.F32, None, 6 * a, 7 * a, 1 << 50, None) == abi.JH_ERR_INVALID
        assert b"too large" in hip.lib().jh_last_error()
        assert hip.lib().jh_op_linear_backward_workspace(rows, n, k, act) == 0
    assert hip.lib().jh_op_gated_ffn_backward(abi.BF16, 2 * a, 8, a, n, 3 * a, k, rows, 4 * a, 8, k, abi.ACT_GELU, 5 * a, k,
                                              abi.F32, None, 7 * a, 1 << 50, None) == abi.JH_ERR_INVALID


@pytest.mark.parametrize("change", [
    dict(product=4), dict(product=-1), dict(t=abi.F32), dict(out=abi.F16), dict(n=12), dict(n=0), dict(k=4),
    dict(rows=(1 << 30) + 1), dict(product=abi.PRODUCT_DX, out=abi.F32), dict(product=abi.PRODUCT_GATED, out=abi.F32),
    dict(product=abi.PRODUCT_DW, t=abi.E4M3, k=64), dict(launches=None),
])
def test_plan_refusals(change):
    base = dict(product=abi.PRODUCT_LINEAR, t=abi.BF16, out=abi.BF16, rows=100, n=64, k=64,
                launches=(hip.LinearLaunch * 2)())
    assert hip.lib().jh_op_linear_plan(*base.values()) == abi.JH_OK
    assert hip.lib().jh_op_linear_plan(*{**base, **change}.values()) == abi.JH_ERR_INVALID


@pytest.mark.parametrize("args", [("dy", BF16, 8, 8, 8), ("linear", torch.int8, 8, 8, 8), ("linear", BF16, 8, 8, 8, torch.int8),
                                  ("linear", BF16, 8, 12, 8), ("dw", E4M3, 16, 16, 16)])
def test_plan_refusals_in_python(args):
    with pytest.raises(hip.HipError) as e:
        hip.linear_plan(*args)
    assert e.value.code == abi.JH_ERR_INVALID


@pytest.mark.parametrize("n,k", [(1024, 1024), (1024, 4096), (4096, 1024), (2304, 768), (4096, 4096), (264, 5000)])
def test_a_contraction_is_planned_by_its_steps(n, k):
    """dw's contraction runs in steps of 64 rows, whose number decides the kernel and the parts; no other border does."""
    for step in range(1, 520):
        plans = {tuple(hip.linear_plan("dw", BF16, 64 * step - i, n, k)) for i in (63, 40, 1, 0)}
        assert len(plans) == 1, (step, plans)


TYPES = {"half": (BF16, None), "e4m3": (E4M3, None), "e4m3 to f32": (E4M3, F32)}


@pytest.mark.parametrize("product,types", list(ROUTES))
def test_sizes_of_every_route(product, types):
    """The sizes that other tests take for a kernel run on it, in both 16-bit types."""
    dtype, out = TYPES[types]
    for name, size in ROUTES[product, types].items():
        assert route(hip.linear_plan(product, dtype, *size, out)) == name, (name, size)
        if types == "half":
            assert route(hip.linear_plan(product, F16, *size, F32 if product in ("linear", "dw") else None)) == name


@pytest.mark.parametrize("product,types", list(ROUTES))
def test_no_other_route(product, types):
    """Sizes drawn over the whole range (up to what a card trains on) take none that is not listed."""
    dtype, out = TYPES[types]
    rng = random.Random(5)

    def draw(lo, hi, step):
        return max(step, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)

    for _ in range(6000):
        size = draw(1, 40000, 1), draw(8, 9000, 8), draw(16, 9000, 16)
        assert route(hip.linear_plan(product, dtype, *size, out)) in ROUTES[product, types], size


def test_norm_gradient_workgroups_fit_the_gpu():
    """A part of dw per workgroup that the 256 CUs hold at once: two each up to 8192 columns, one of longer rows."""
    for hidden, most in ((8, 512), (2056, 512), (8192, 512), (8200, 256), (16384, 256)):
        assert hip.rms_norm_backward_workspace(100000, hidden) == most * hidden * 4
    assert hip.rms_norm_backward_workspace(200, 16384) == 200 * 16384 * 4
