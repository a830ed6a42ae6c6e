"""Arguments that the feed-forward operators refuse, and their workspace sizes: checked on the host before anything is
launched, so no device is needed (addresses are made up and never read)."""
import pytest

from julia1_amd import abi, hip

A = 1 << 30  # made-up 16-byte aligned addresses, far apart
STEP = 1 << 28


def at(i):
    return A + i * STEP


def refused(fn, base, **change):
    """`base` is a call's arguments by name, in order; with `change` the call must be refused as invalid."""
    bad = {k: v for k, v in change.items() if k not in base}
    assert not bad, bad
    args = {**base, **change}
    assert fn(*args.values()) == abi.JH_ERR_INVALID, change
    return hip.lib().jh_last_error().decode()


NORM = dict(xt=abi.BF16, x=at(0), ldx=64, rt=abi.F32, r=at(1), ldr=64, ro=at(2), ldro=64, rows=4, h=64, w=at(3),
            eps=1e-6, ot=abi.E4M3, out=at(4), ldo=64, scales=at(5), rstd=at(6), stream=None)


@pytest.mark.parametrize("change", [
    dict(xt=abi.E4M3), dict(xt=7), dict(rt=abi.F16), dict(ot=abi.F32), dict(ot=abi.F16), dict(h=0), dict(h=60),
    dict(h=16392, ldx=16392), dict(eps=-1.0), dict(eps=float("nan")), dict(r=None), dict(ro=None), dict(w=None),
    dict(x=None), dict(x=at(0) + 8), dict(ldx=56), dict(ldx=68), dict(ldr=66), dict(out=None), dict(out=at(4) + 4),
    dict(ldo=68), dict(ldo=56), dict(scales=None), dict(ot=abi.BF16), dict(out=at(0)), dict(out=at(1)),
    dict(ro=at(0)), dict(ro=at(1), ldro=128), dict(rstd=at(5)), dict(scales=at(3)), dict(rows=1 << 31),
    dict(ldx=1 << 22),
])
def test_rms_norm_refusals(change):
    assert refused(hip.lib().jh_op_rms_norm, NORM, **change)


NORM_B = dict(yt=abi.BF16, dy=at(0), ldy=64, st=abi.F32, s=at(1), lds=64, rows=4, h=64, w=at(2), rstd=at(3),
              dt=abi.F32, dres=at(4), ldr=64, ds=at(5), ldd=64, dw=at(6), ws=at(7), wsb=1 << 20, stream=None)


@pytest.mark.parametrize("change", [
    dict(yt=abi.E4M3), dict(st=abi.F16), dict(dt=abi.F16), dict(h=4), dict(w=None), dict(rstd=None), dict(dy=None),
    dict(s=None), dict(ds=None), dict(ws=None), dict(ws=at(7) + 4), dict(wsb=64 * 4 - 1), dict(ds=at(0)),
    dict(ds=at(4), ldd=128), dict(dw=at(2)), dict(ws=at(5)), dict(dw=at(7)),
])
def test_rms_norm_backward_refusals(change):
    assert refused(hip.lib().jh_op_rms_norm_backward, NORM_B, **change)


def test_rms_norm_backward_needs_w_without_rows_too():
    """dw of no rows is zeros, from a kernel that reads w before it knows."""
    refused(hip.lib().jh_op_rms_norm_backward, NORM_B, rows=0, w=None)


QUANT = dict(xt=abi.F32, x=at(0), ldx=64, rows=4, n=64, q=at(1), ldq=64, scales=at(2), stream=None)


@pytest.mark.parametrize("change", [
    dict(xt=abi.E4M3), dict(n=0), dict(n=63), dict(n=16400, ldx=16400, ldq=16400), dict(x=None), dict(q=None),
    dict(scales=None), dict(ldx=66), dict(ldq=60), dict(q=at(1) + 4), dict(q=at(0)), dict(scales=at(1)),
])
def test_quantize_rows_refusals(change):
    assert refused(hip.lib().jh_op_quantize_rows, QUANT, **change)


LINEAR = dict(t=abi.BF16, x=at(0), ldx=64, xs=None, rows=4, w=at(1), ws=None, n=32, k=64, bias=at(2), act=0,
              resid=at(3), ldr=32, ot=abi.F32, out=at(4), ldo=32, pre=at(5), ldp=32, stream=None)


@pytest.mark.parametrize("change", [
    dict(t=abi.F32), dict(t=9), dict(n=0), dict(n=36), dict(k=0), dict(k=60), dict(act=5), dict(act=-1),
    dict(ot=abi.F16), dict(ot=abi.E4M3), dict(xs=at(6)), dict(ws=at(6)), dict(x=None), dict(w=None), dict(out=None),
    dict(x=at(0) + 2), dict(ldx=56), dict(ldx=70), dict(ldr=24), dict(ldr=34), dict(ldo=30), dict(ldp=36),
    dict(out=at(0)), dict(out=at(1)), dict(pre=at(4)), dict(pre=at(3)), dict(out=at(3), ldo=64), dict(rows=1 << 31),
    dict(n=1 << 23), dict(t=abi.E4M3), dict(t=abi.E4M3, pre=None, k=24, ldx=32), dict(ldx=1 << 22),
    dict(t=abi.E4M3, pre=None, ot=abi.F16),
])
def test_linear_refusals(change):
    assert refused(hip.lib().jh_op_linear, LINEAR, **change)


def test_outputs_over_the_bias_or_a_scale_are_refused():
    e4m3 = dict(LINEAR, t=abi.E4M3, pre=None, xs=at(6), ws=at(7), ot=abi.BF16)
    gated = dict(GATED, t=abi.E4M3, gu=None, xs=at(6), ws=at(7), ldx=64)
    for change in (dict(bias=at(4)), dict(xs=at(4) + 16), dict(ws=at(4) + 64)):
        refused(hip.lib().jh_op_linear, e4m3, **change)
    refused(hip.lib().jh_op_linear, LINEAR, bias=at(5) + 32)
    for change in (dict(xs=at(2)), dict(ws=at(2) - 24 * 4)):  # the up half's scales
        refused(hip.lib().jh_op_gated_ffn, gated, **change)


def test_linear_in_place_residual_is_not_refused():
    """resid may be out: with no rows such a call does nothing (and needs no device)."""
    args = {**LINEAR, "rows": 0, "out": at(3)}
    assert hip.lib().jh_op_linear(*args.values()) == abi.JH_OK


LINEAR_B = dict(t=abi.BF16, dy=at(0), ldy=32, x=at(1), ldx=64, rows=4, w=at(2), n=32, k=64, act=abi.ACT_GELU,
                pre=at(3), ldp=32, dx=at(4), ldd=64, gt=abi.F32, dw=at(5), db=at(6), ws=at(7), wsb=1 << 26, stream=None)


@pytest.mark.parametrize("change", [
    dict(t=abi.E4M3, gt=abi.E4M3), dict(t=abi.F32), dict(gt=abi.F16), dict(act=6), dict(n=20), dict(k=12), dict(pre=None), dict(x=None),
    dict(w=None), dict(dy=None), dict(dx=None, dw=None, db=None), dict(ws=None), dict(ws=at(7) + 8), dict(wsb=255),
    dict(ldy=24), dict(ldd=60), dict(dx=at(0)), dict(dw=at(2)), dict(db=at(5)), dict(ws=at(3)), dict(dx=at(7)),
])
def test_linear_backward_refusals(change):
    assert refused(hip.lib().jh_op_linear_backward, LINEAR_B, **change)


GATED = dict(t=abi.F16, x=at(0), ldx=64, xs=None, rows=4, wi=at(1), ws=None, inter=24, k=64, act=abi.ACT_SILU,
             out=at(2), ldo=24, gu=at(3), ldg=48, stream=None)


@pytest.mark.parametrize("change", [
    dict(t=abi.F32), dict(t=abi.E4M3), dict(inter=20), dict(inter=0), dict(k=4), dict(act=7), dict(x=None),
    dict(wi=None), dict(out=None), dict(ldo=16), dict(ldg=40), dict(out=at(1) + 24 * 64 * 2), dict(gu=at(0)),
    dict(gu=at(2)), dict(xs=at(5)), dict(inter=1 << 20, k=2048, ldx=2048, ldo=1 << 20, ldg=1 << 21),
])
def test_gated_refusals(change):
    assert refused(hip.lib().jh_op_gated_ffn, GATED, **change)


GATED_B = dict(t=abi.F16, dh=at(0), ldh=24, gu=at(1), ldg=48, x=at(2), ldx=64, rows=4, wi=at(3), inter=24, k=64,
               act=abi.ACT_SILU, dx=at(4), ldd=64, gt=abi.F16, dwi=at(5), ws=at(6), wsb=1 << 26, stream=None)


@pytest.mark.parametrize("change", [
    dict(t=abi.E4M3, gt=abi.E4M3), dict(gt=abi.BF16), dict(inter=12), dict(act=9), dict(gu=None), dict(dh=None), dict(x=None),
    dict(wi=None), dict(dx=None, dwi=None), dict(ws=None), dict(wsb=100), dict(ldg=24), dict(ldh=16),
    dict(dx=at(2)), dict(dwi=at(3)), dict(ws=at(1)), dict(inter=1 << 22),
])
def test_gated_backward_refusals(change):
    assert refused(hip.lib().jh_op_gated_ffn_backward, GATED_B, **change)


def test_host_tensors_are_refused():
    """The Python calls take tensors of the current device alone: an address of host memory would fault there."""
    torch = pytest.importorskip("torch")
    x, w, out = torch.zeros(4, 64), torch.zeros(32, 64), torch.zeros(4, 32)
    for call in (lambda: hip.op_linear(x, w, out), lambda: hip.op_gated_ffn(x, w, out[:, :16]),
                 lambda: hip.op_rms_norm(x, torch.ones(64), 1e-6, x.bfloat16()),
                 lambda: hip.op_quantize_rows(x, torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4)),
                 lambda: hip.op_rms_norm_backward(x, x, torch.ones(64), torch.ones(4), x.clone()),
                 lambda: hip.op_linear_backward(out, x, w, None, dx=x), lambda: hip.op_gated_ffn_backward(
                     out[:, :16], out, x, w, None, dx=x)):
        with pytest.raises(hip.HipError) as e:
            call()
        assert e.value.code == abi.JH_ERR_INVALID and "current device" in str(e.value)


def test_column_ranges_of_one_buffer_that_share_a_column():
    """Ranges of one buffer's columns that share one are refused, also where a range wraps onto the next row."""
    base = dict(LINEAR, resid=None, pre=None, bias=None, ot=abi.BF16, x=at(0), ldx=256, ldo=256, n=32)
    refused(hip.lib().jh_op_linear, base, out=at(0) + 2 * 48)      # columns 48 .. 79 over x's 0 .. 63
    refused(hip.lib().jh_op_linear, base, out=at(0) + 2 * 240)     # 240 .. 271 wrap onto the next row's first


def test_workspace_sizes():
    assert hip.rms_norm_backward_workspace(1, 64) == 64 * 4
    assert hip.rms_norm_backward_workspace(100000, 4096) == 512 * 4096 * 4
    for rows in (2**31 - 4, 2**31 - 1):  # the number of workgroups is formed without passing 31 bits
        assert hip.rms_norm_backward_workspace(rows, 64) == 512 * 64 * 4
    assert hip.linear_backward_workspace(4, 32, 64, "none") < hip.linear_backward_workspace(4, 32, 64, "gelu") + 1
    # the gradient before the activation always has its place
    assert hip.linear_backward_workspace(5000, 1024, 512, "silu") >= 5000 * 1024 * 2
    assert hip.gated_ffn_backward_workspace(5000, 1024, 512) >= 5000 * 2048 * 2
    for fn, args in ((hip.rms_norm_backward_workspace, (4, 12)), (hip.linear_backward_workspace, (4, 30, 64)),
                     (hip.linear_backward_workspace, (4, 32, 64, "tanh")), (hip.gated_ffn_backward_workspace, (4, 12, 64))):
        with pytest.raises(hip.HipError):
            fn(*args)
