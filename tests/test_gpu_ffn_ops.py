"""The feed-forward operators (RMS norm, row quantisation, linear layers, gated projections) on the GPU against their
definitions in 64 bits on the same inputs.

Tolerances are worst-case bounds, element by element: a rounding to type t is off by at most finfo(t).eps / 2 of the
value (and half the smallest step of f16 near zero); a sum of k products whose magnitudes add up to S is off by at most
k 2^-23 S; an activation's value or slope at z is off by at most (1 + |z|) 2^-19 (erf's approximation is within 1e-6, the
hardware's exponential and reciprocal within 2^-22 of theirs); activations' slopes are at most 1.2.  With e4m3 operands
and a bf16 output the MFMA aligns the products to the largest and may drop 2^-13 of it from each.  e4m3 codes and whole
numbers are equal."""
import math

import pytest

torch = pytest.importorskip("torch")

from julia1_amd import abi, hip  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
EPS = 1e-6
ACT = 2.0**-19


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * std


def half(t):
    return torch.finfo(t).eps / 2


def floor(t):
    return 2.0**-25 if t == F16 else 0.0


class Padded:
    """A matrix inside a larger buffer of sentinels: `t` is the view, check() that nothing around it was written."""

    def __init__(self, rows, cols, dtype, pad=16, fill=-7.0):
        self.buf = torch.full((rows + 2, cols + pad), fill, device="cuda", dtype=F32).to(dtype)
        self.t = self.buf[1:rows + 1, :cols]
        self.fill = fill

    def check(self):
        b = self.buf.float()
        rows, cols = self.t.shape
        assert bool((b[0] == self.fill).all()) and bool((b[rows + 1:] == self.fill).all())
        assert bool((b[:, cols:] == self.fill).all())


def padded_like(v, dtype, pad=16):
    """`v` in rows with NaN behind them, which must not be read into any result."""
    buf = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), device="cuda", dtype=F32).to(dtype)
    buf[:, :v.shape[1]] = v.to(dtype)
    return buf[:, :v.shape[1]]


def close(got, want, tol, name):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (name, int(bad.sum()), float((got.double() - want).abs().max()),
                                 bad.nonzero()[:4].tolist())


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z**3))
        return z / 2 * (1 + t), (1 + t) / 2 + z / 2 * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def nearest_e4m3(v):
    """The nearest e4m3 value, ties to the even code (|v| <= 448)."""
    step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4)
    return torch.round(v / step) * step


# ---------------------------------------------------------------- RMS norm, row quantisation

NORMS = [(BF16, F32, BF16), (BF16, BF16, E4M3), (F16, F16, F16), (F16, F32, E4M3), (F32, F32, F16), (F32, F32, E4M3),
         (BF16, None, BF16), (F32, None, E4M3)]
# one chunk of one lane, a ragged last chunk, each register count per lane, both row owners (a wave, a workgroup)
WIDTHS = [(1, 8), (5, 120), (3, 520), (70, 768), (9, 1024), (2, 1536), (6, 2048), (3, 2056), (5, 5000), (2, 8192),
          (1, 9000), (3, 16384)]


def norm_inputs(g, rows, h, xt, rt):
    x = randn(g, rows, h)
    resid = None
    if rt is not None:
        resid = randn(g, rows, h, std=2.0)
        resid[:, :: max(1, h // 5)] *= 30
        resid = resid.to(rt)
    return x.to(xt), resid, 1 + randn(g, h, std=0.3)


@pytest.mark.parametrize("rows,h", WIDTHS)
@pytest.mark.parametrize("xt,rt,ot", NORMS)
def test_rms_norm(rows, h, xt, rt, ot):
    g = gen(rows * h)
    x, resid, w = norm_inputs(g, rows, h, xt, rt)
    if rows > 2:
        x[1] = 0
        if resid is not None:
            resid[1] = 0
    x = padded_like(x, xt)
    out, rstd = Padded(rows, h, ot), torch.empty(rows, device="cuda")
    kw = {}
    s = x
    if resid is not None:
        so = Padded(rows, h, rt)
        kw.update(resid=resid, resid_out=so.t)
        s = (x.float() + resid.float()).to(rt)
    if ot == E4M3:
        kw.update(scales=torch.empty(rows, device="cuda"))
    hip.op_rms_norm(x, w, EPS, out.t, rstd=rstd, **kw)
    torch.cuda.synchronize()
    out.check()
    if resid is not None:
        so.check()
        assert torch.equal(so.t, s)
    s, w = s.double(), w.double()
    r = 1 / torch.sqrt((s * s).mean(dim=1) + EPS)
    rel = (h / 2 + 16) * 2.0**-24
    close(rstd, r, rel * r, "rstd")
    y = s * r[:, None] * w
    if ot != E4M3:
        close(out.t, y, y.abs() * (half(ot) + 2 * rel) + floor(ot), "out")
        return
    p = s * w
    top = p.abs().amax(dim=1)
    close(kw["scales"], y.abs().amax(dim=1) / 448, 2 * rel * y.abs().amax(dim=1) / 448, "scales")
    want = nearest_e4m3(p * 448 / torch.where(top > 0, top, 1.0)[:, None])
    assert torch.equal(out.t.double(), want)


def test_rms_norm_in_place():
    g = gen(3)
    x, resid, w = norm_inputs(g, 33, 5000, BF16, F32)
    a, b = torch.empty(33, 5000, device="cuda", dtype=BF16), torch.empty(33, 5000, device="cuda", dtype=BF16)
    apart = torch.empty_like(resid)
    hip.op_rms_norm(x, w, EPS, a, resid=resid, resid_out=apart)
    hip.op_rms_norm(x, w, EPS, b, resid=resid, resid_out=resid)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(apart, resid)


@pytest.mark.parametrize("xt", [BF16, F16, F32])
@pytest.mark.parametrize("rows,h", WIDTHS)
def test_quantize_rows(rows, h, xt):
    g = gen(rows + h)
    x = randn(g, rows, h)
    x[0, : h // 2] *= 2.0**-7   # codes of the smallest steps
    if rows > 2:
        x[2] = 0
    x = padded_like(x, xt)
    q, scales = Padded(rows, h, E4M3), torch.empty(rows, device="cuda")
    hip.op_quantize_rows(x, q.t, scales)
    torch.cuda.synchronize()
    q.check()
    v = x.double()
    top = v.abs().amax(dim=1)
    close(scales, top / 448, top / 448 * half(F32), "scales")
    assert torch.equal(q.t.double(), nearest_e4m3(v * 448 / torch.where(top > 0, top, 1.0)[:, None]))


def test_quantize_ties_and_not_numbers():
    """Exact ties go to the even code, for every pair of neighbouring codes; a NaN stays one and leaves its row's other
    codes alone; an infinity leaves its row no finite scale."""
    codes = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    ties = (codes[:-1] + codes[1:]) / 2
    row = torch.cat([ties, -ties, codes[:4]]).cuda()
    row[-1] = 448.0
    x = torch.stack([row, row * 3, row, row]).float()
    x[2, 5], x[3, 7] = float("nan"), float("inf")
    q, scales = torch.empty(4, 256, device="cuda", dtype=E4M3), torch.empty(4, device="cuda")
    hip.op_quantize_rows(x, q, scales)
    torch.cuda.synchronize()
    want = nearest_e4m3(row)
    assert torch.equal(q[0].double(), want) and torch.equal(q[1].double(), want)
    assert scales[:3].tolist() == [1.0, 3.0, 1.0] and not math.isfinite(scales[3].item())
    rest = torch.arange(256, device="cuda") != 5
    assert math.isnan(q[2, 5].float().item()) and torch.equal(q[2][rest].double(), want[rest])


@pytest.mark.parametrize("dt,st,gt", [(BF16, BF16, BF16), (BF16, F32, F32), (BF16, BF16, F32), (F16, F32, F16),
                                      (F32, F32, F32)])
@pytest.mark.parametrize("rows,h", WIDTHS + [(2100, 264), (1500, 4096)])
def test_rms_norm_backward(rows, h, dt, st, gt):
    g = gen(rows + 3 * h)
    s = randn(g, rows, h, std=2.0).to(st)
    dy, dres, w = randn(g, rows, h).to(dt), randn(g, rows, h).to(gt), 1 + randn(g, h, std=0.3)
    rstd = (1 / torch.sqrt(s.double().square().mean(dim=1) + EPS)).float()
    ds, dw = Padded(rows, h, gt), torch.full((h,), float("nan"), device="cuda")
    ws = torch.empty(hip.rms_norm_backward_workspace(rows, h), dtype=torch.uint8, device="cuda")
    hip.op_rms_norm_backward(padded_like(dy, dt), padded_like(s, st), w, rstd, ds.t, dw, ws, dres=dres)
    plain = torch.empty(rows, h, device="cuda", dtype=gt)
    hip.op_rms_norm_backward(dy, s, w, rstd, plain)  # no residual gradient, no dw
    torch.cuda.synchronize()
    ds.check()
    r, n, gy = rstd.double()[:, None], s.double() * rstd.double()[:, None], dy.double() * w.double()
    along, size = (gy * n).mean(dim=1, keepdim=True), (gy * n).abs().mean(dim=1, keepdim=True)
    want = r * (gy - n * along)
    tol = r * (gy.abs() * 8 + n.abs() * size * (h + 16)) * 2.0**-24
    close(plain, want, tol + want.abs() * half(gt) + floor(gt), "ds alone")
    want = want + dres.double()
    close(ds.t, want, tol + (want.abs() + dres.double().abs() * 2.0**-16) * half(gt) + want.abs() * 2.0**-23 + floor(gt),
          "ds")
    t = dy.double() * n
    close(dw, t.sum(dim=0), t.abs().sum(dim=0) * (rows + 16) * 2.0**-24, "dw")


def test_rms_norm_backward_in_place_and_no_rows():
    g = gen(8)
    s, dy, w = randn(g, 40, 2056).to(BF16), randn(g, 40, 2056).to(BF16), 1 + randn(g, 2056, std=0.3)
    rstd = (1 / torch.sqrt(s.double().square().mean(dim=1) + EPS)).float()
    ws = torch.empty(hip.rms_norm_backward_workspace(40, 2056), dtype=torch.uint8, device="cuda")
    want, dw = torch.empty_like(s), torch.empty(2056, device="cuda")
    hip.op_rms_norm_backward(dy, s, w, rstd, want, dw, ws, dres=dy)
    for place in ("dy", "s"):
        a, b, again = dy.clone(), s.clone(), torch.empty(2056, device="cuda")
        hip.op_rms_norm_backward(a, b, w, rstd, a if place == "dy" else b, again, ws, dres=dy)
        torch.cuda.synchronize()
        assert torch.equal(a if place == "dy" else b, want) and torch.equal(dw, again)
    d = dy.clone()
    hip.op_rms_norm_backward(dy, s, w, rstd, d, dres=d)
    torch.cuda.synchronize()
    assert torch.equal(d, want)
    hip.op_rms_norm_backward(dy[:0], s[:0], w, rstd[:0], want[:0], dw, ws)
    torch.cuda.synchronize()
    assert torch.equal(dw, torch.zeros_like(dw))


# ---------------------------------------------------------------- linear layers and gated projections

def operands(g, rows, n, k, t):
    """x, w in type t inside padded rows (w without padding), their scales, and both in 64 bits."""
    x, w = randn(g, rows, k), randn(g, n, k, std=1 / math.sqrt(k))
    if t != E4M3:
        x, w = padded_like(x, t), w.to(t)
        return x, w, {}, x.double(), w.double()
    xs, ws = 0.5 + torch.rand(rows, device="cuda", generator=g), 0.5 + torch.rand(n, device="cuda", generator=g)
    x, w = padded_like(x * 4, t), (w * 64).to(t)
    return (x, w, dict(x_scale=xs, w_scale=ws), x.double() * xs.double()[:, None], w.double() * ws.double()[:, None])


def product_tol(x, w, k, e4m3_bf16):
    tol = (x.abs() @ w.abs().t()) * (k + 4) * 2.0**-23
    if e4m3_bf16:
        tol = tol + k * 2.0**-13 * x.abs().amax(dim=1)[:, None] * w.abs().amax(dim=1)
    return tol


# (rows, n, k): one token; both sides of 16, 32 and 64 rows; tiles that end inside rows, columns and K steps; one K
# step and less; several tiles each way
SIZES = [(1, 8, 16), (1, 768, 1152), (16, 264, 80), (17, 72, 1000), (33, 768, 64), (64, 520, 144), (65, 136, 208),
         (127, 128, 8 * 26), (129, 264, 1152), (300, 1000, 400), (513, 2312, 768), (1100, 776, 1040)]


def linear_case(rows, n, k, t, out_t, act, with_bias, with_resid, with_pre, seed):
    if t == E4M3:
        k = (k + 15) // 16 * 16
    g = gen(seed)
    x, w, scales, x64, w64 = operands(g, rows, n, k, t)
    bias = randn(g, n + 1)[1:] if with_bias else None       # 4-byte aligned only
    if bias is not None:
        bias = torch.as_strided(bias, (n,), (1,))
    resid = padded_like(randn(g, rows, n, std=2.0), out_t) if with_resid else None
    out, pre = Padded(rows, n, out_t), Padded(rows, n, t) if with_pre else None
    hip.op_linear(x, w, out.t, bias=bias, act=act, resid=resid, pre=None if pre is None else pre.t, **scales)
    torch.cuda.synchronize()
    out.check()
    z, tz = x64 @ w64.t(), product_tol(x64, w64, k, t == E4M3 and out_t == BF16)
    if bias is not None:
        z, tz = z + bias.double(), tz + (z.abs() + bias.double().abs()) * 2.0**-23
    if pre is not None:
        pre.check()
        close(pre.t, z, tz + z.abs() * half(t) + floor(t), "pre")
    y = act64(z, act)[0]
    ty = 1.2 * tz + (0 if act in ("none", "relu") else 1) * z.abs() * (1 + z.abs()) * ACT
    if resid is not None:
        y, ty = y + resid.double(), ty + (y.abs() + resid.double().abs()) * 2.0**-23
    close(out.t, y, ty * (1 + 2 * half(out_t)) + y.abs() * half(out_t) + floor(out_t), "out")
    assert float((out.t.double() - y).norm() / y.norm()) < half(out_t) * (1 if out_t != F32 else 64)


@pytest.mark.parametrize("rows,n,k", SIZES)
@pytest.mark.parametrize("t,out_t", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (E4M3, BF16), (E4M3, F32)])
def test_linear(rows, n, k, t, out_t):
    """Every size and type; the epilogue's parts alternate with the size, all at once among them."""
    i = SIZES.index((rows, n, k))
    linear_case(rows, n, k, t, out_t, ["gelu", "none", "silu", "relu", "gelu_tanh"][i % 5], i % 2 == 0, i % 3 != 1,
                t != E4M3 and i % 4 < 2, seed=100 + i)


# sizes for each kernel that larger products run on: 128 x 128 tiles one to a CU and two to a CU, 128 x 256 tiles, 256 x 256
# tiles, those for whole rounds of the CUs with the rest on smaller ones, and 64 x 64 tiles of a long contraction
KERNELS = [(1000, 4000, 520), (1500, 4000, 520), (1600, 4704, 520), (1500, 4000, 2080), (3900, 4000, 520),
           (4700, 4000, 520), (129, 264, 4104)]


@pytest.mark.parametrize("rows,n,k", KERNELS)
@pytest.mark.parametrize("t,out_t", [(BF16, BF16), (F16, F32), (E4M3, BF16), (E4M3, F32)])
def test_linear_kernels(rows, n, k, t, out_t):
    linear_case(rows, n, k, t, out_t, "silu", True, True, t != E4M3, seed=rows)


@pytest.mark.parametrize("rows,n,k", KERNELS)
@pytest.mark.parametrize("t", [BF16, F16, E4M3])
def test_gated_ffn_kernels(rows, n, k, t):
    test_gated_ffn(rows, n // 16 * 8, k, t)


# the same for both gradients (dx: rows x k over n; dw: n x k over rows), contractions that are cut into parts, and 64 x 64
# tiles whose waves share a long contraction
@pytest.mark.parametrize("rows,n,k", [(1500, 520, 4000), (3900, 520, 4000), (4700, 520, 4000), (520, 1504, 4000),
                                      (520, 3904, 4000), (520, 4704, 4000), (9000, 1032, 776), (264, 6008, 264),
                                      (1000, 3600, 1000), (3600, 1000, 1000), (7000, 1032, 776)])
@pytest.mark.parametrize("t,grad_t", [(BF16, BF16), (F16, F32)])
def test_linear_backward_kernels(rows, n, k, t, grad_t):
    test_linear_backward(rows, n, k, t, grad_t, "gelu")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 200])
def test_linear_activations(act, rows):
    linear_case(rows, 136, 256, BF16, F32, act, True, True, True, seed=7)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [4, 60])
def test_activations_of_large_values(act, rows):
    """Values whose squares pass FP32's range: each activation is z or 0 there, its slope 1 or 0 (z^2 itself is inf)."""
    n, k = 32, 16
    z = torch.tensor([1e18, 3e19, 2e30, 1e38], device="cuda").repeat_interleave(8)[None, :].repeat(rows, 1)
    z[1::2] *= -1
    x = torch.zeros(rows, k, device="cuda", dtype=BF16)
    out, pre, h = (torch.empty(rows, n, device="cuda", dtype=BF16) for _ in range(3))
    hip.op_linear(x, torch.zeros(n, k, device="cuda", dtype=BF16), out, bias=z[0].abs().contiguous(), act=act, pre=pre)
    torch.cuda.synchronize()
    assert torch.equal(pre, z.abs().to(BF16)) and torch.equal(out, pre)
    x[:, 0] = z[:, 0].sign().to(BF16)
    wi = torch.zeros(2 * n, k, device="cuda", dtype=BF16)
    wi[:n, 0], wi[n:, 0] = z[0].to(BF16), x[0, 0]
    hip.op_gated_ffn(x, wi, h, act=act)
    want = torch.where((z > 0) | (act == "none"), z.abs(), torch.zeros_like(z)).to(BF16)
    torch.cuda.synchronize()
    assert torch.equal(h, want)
    pre = z.to(BF16)
    dy, db = torch.ones(rows, n, device="cuda", dtype=BF16), torch.empty(n, device="cuda")
    ws = torch.empty(hip.gated_ffn_backward_workspace(rows, n, k) + hip.linear_backward_workspace(rows, n, k, act),
                     dtype=torch.uint8, device="cuda")
    hip.op_linear_backward(dy, x, wi[:n], ws, act=act, pre=pre, dbias=db)
    dwi = torch.empty(2 * n, k, device="cuda")
    hip.op_gated_ffn_backward(dy, torch.cat([pre, dy], dim=1), x, wi, ws, act=act, dw=dwi)
    torch.cuda.synchronize()
    slope = torch.where((z > 0) | (act == "none"), 1.0, 0.0)
    assert torch.equal(db, slope.sum(dim=0))
    assert torch.equal(dwi[:n, 0], (slope * z.sign()).sum(dim=0))


def test_linear_residual_in_place():
    g = gen(5)
    for rows in (4, 150):
        x, w, resid = randn(g, rows, 256).to(BF16), randn(g, 392, 256, std=0.06).to(BF16), randn(g, rows, 392)
        apart = torch.empty_like(resid)
        hip.op_linear(x, w, apart, resid=resid, act="silu")
        hip.op_linear(x, w, resid, resid=resid, act="silu")
        torch.cuda.synchronize()
        assert torch.equal(apart, resid)


def test_linear_column_ranges_of_one_buffer():
    """x and out as column ranges of one buffer, as a caller with a packed workspace holds them."""
    g = gen(6)
    buf = randn(g, 140, 64 + 200).to(BF16)
    x, out, w = buf[:, :64], buf[:, 64:], randn(g, 200, 64, std=0.1).to(BF16)
    apart = torch.empty(140, 200, device="cuda", dtype=BF16)
    keep = x.clone()
    hip.op_linear(x, w, apart)
    hip.op_linear(x, w, out)
    torch.cuda.synchronize()
    assert torch.equal(out, apart) and torch.equal(x, keep)


@pytest.mark.parametrize("rows", [5, 70])
def test_linear_not_a_number_stays_in_its_row_and_column(rows):
    """A NaN row of x spoils its output row, a NaN row of W its output column, and nothing else; relu passes it on."""
    g = gen(9)
    x, w = randn(g, rows, 136).to(BF16), randn(g, 72, 136, std=0.1).to(BF16)
    clean, out = torch.empty(rows, 72, device="cuda"), torch.empty(rows, 72, device="cuda")
    hip.op_linear(x, w, clean, act="relu")
    x[2, 135] = float("nan")
    w[40, 3] = float("inf")
    hip.op_linear(x, w, out, act="relu")
    torch.cuda.synchronize()
    assert bool(out[2].isnan().all())
    keep = torch.ones(rows, 72, dtype=torch.bool, device="cuda")
    keep[2], keep[:, 40] = False, False
    assert torch.equal(out[keep], clean[keep]) and not bool(out[:, 40][x[:, 3] > 0].isfinite().any())


def test_linear_no_rows():
    x, w = torch.empty(0, 64, device="cuda", dtype=BF16), torch.empty(32, 64, device="cuda", dtype=BF16)
    hip.op_linear(x, w, torch.empty(0, 32, device="cuda", dtype=BF16))
    hip.op_gated_ffn(x, w, torch.empty(0, 16, device="cuda", dtype=BF16))
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,n,k", [(s[0], max(8, s[1] // 16 * 8), s[2]) for s in SIZES])
@pytest.mark.parametrize("t", [BF16, F16, E4M3])
def test_gated_ffn(rows, n, k, t):
    if t == E4M3:
        k = (k + 15) // 16 * 16
    g = gen(rows + n + k)
    x, wi, scales, x64, w64 = operands(g, rows, 2 * n, k, t)
    out_t = BF16 if t == E4M3 else t
    act = ["gelu", "silu", "gelu_tanh", "relu"][(rows + k) % 4]
    out, gu = Padded(rows, n, out_t), Padded(rows, 2 * n, out_t) if t != E4M3 and rows != 33 else None
    hip.op_gated_ffn(x, wi, out.t, act=act, gu=None if gu is None else gu.t, **scales)
    torch.cuda.synchronize()
    out.check()
    z, tz = x64 @ w64.t(), product_tol(x64, w64, k, t == E4M3)
    if gu is not None:
        gu.check()
        close(gu.t, z, tz + z.abs() * half(t) + floor(t), "gu")
    (a, _), u = act64(z[:, :n], act), z[:, n:]
    ta = 1.2 * tz[:, :n] + z[:, :n].abs() * (1 + z[:, :n].abs()) * ACT
    tol = ta * (u.abs() + tz[:, n:]) + a.abs() * tz[:, n:] + (a * u).abs() * 2.0**-23
    close(out.t, a * u, tol * 1.01 + (a * u).abs() * half(out_t) + floor(out_t), "out")


GRADS = [(1, 8, 16), (5, 72, 264), (64, 136, 128), (130, 264, 200), (700, 520, 392), (1537, 1024, 136), (3000, 64, 72)]


def product_bounds(dz, tdz, w, x, t, grad_t):
    """dx = dz w and dw = dz^T x with their tolerances, for dz off by at most tdz before its rounding to t."""
    e = tdz * (1 + 2 * half(t)) + dz.abs() * half(t) + floor(t)
    n, rows = w.shape[0], x.shape[0]
    dx, dw = dz @ w, dz.t() @ x
    tx = e @ w.abs() + (n + 4) * 2.0**-23 * ((dz.abs() + e) @ w.abs())
    tw = e.t() @ x.abs() + (rows + 32) * 2.0**-23 * ((dz.abs() + e).t() @ x.abs())
    return (dx, tx * 1.01 + dx.abs() * half(t) + floor(t)), (dw, tw * 1.01 + dw.abs() * half(grad_t) + floor(grad_t))


@pytest.mark.parametrize("rows,n,k", GRADS)
@pytest.mark.parametrize("t,grad_t,act", [(BF16, BF16, "gelu"), (BF16, F32, "none"), (F16, F16, "silu"),
                                          (F16, F32, "gelu_tanh"), (BF16, F32, "relu")])
def test_linear_backward(rows, n, k, t, grad_t, act):
    g = gen(rows + n + k)
    x, w = padded_like(randn(g, rows, k), t), randn(g, n, k, std=1 / math.sqrt(k)).to(t)
    dy = padded_like(randn(g, rows, n), t)
    pre = padded_like(randn(g, rows, n, std=1.5), t) if act != "none" else None
    dx, dw = Padded(rows, k, t), torch.full((n, k), float("nan"), device="cuda", dtype=grad_t)
    db = torch.full((n,), float("nan"), device="cuda")
    ws = torch.full((hip.linear_backward_workspace(rows, n, k, act) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    hip.op_linear_backward(dy, x, w, ws[:-64], act=act, pre=pre, dx=dx.t, dw=dw, dbias=db)
    torch.cuda.synchronize()
    dx.check()
    assert bool((ws[-64:] == 0xFF).all())
    dz, tdz = dy.double(), torch.zeros(rows, n, device="cuda", dtype=torch.float64)
    if pre is not None:
        z = pre.double()
        dz, tdz = dz * act64(z, act)[1], dz.abs() * (1 + z.abs()) * ACT
    close(db, dz.sum(dim=0), tdz.sum(dim=0) + dz.abs().sum(dim=0) * (rows + 16) * 2.0**-24, "dbias")
    if act == "none":  # dz is dy itself: not rounded again
        (wx, tx), (ww, tw) = product_bounds(dz, tdz, w.double(), x.double(), F32, grad_t)
        tx = tx + wx.abs() * half(t) + floor(t)
    else:
        (wx, tx), (ww, tw) = product_bounds(dz, tdz, w.double(), x.double(), t, grad_t)
    close(dx.t, wx, tx, "dx")
    close(dw, ww, tw, "dw")
    # each gradient alone has the same bits
    a, b, c = torch.empty(rows, k, device="cuda", dtype=t), torch.empty_like(dw), torch.empty_like(db)
    hip.op_linear_backward(dy, x, w, ws[:-64], act=act, pre=pre, dx=a)
    hip.op_linear_backward(dy, x, w, ws[:-64], act=act, pre=pre, dw=b)
    hip.op_linear_backward(dy, x, w, ws[:-64], act=act, pre=pre, dbias=c)
    torch.cuda.synchronize()
    assert torch.equal(a, dx.t) and torch.equal(b, dw) and torch.equal(c, db)


@pytest.mark.parametrize("rows,n,k", GRADS)
@pytest.mark.parametrize("t,grad_t,act", [(BF16, BF16, "gelu"), (F16, F32, "silu"), (BF16, F32, "gelu_tanh")])
def test_gated_ffn_backward(rows, n, k, t, grad_t, act):
    n = max(8, n // 16 * 8)
    g = gen(rows + n + k)
    x, wi = padded_like(randn(g, rows, k), t), randn(g, 2 * n, k, std=1 / math.sqrt(k)).to(t)
    dh, gu = padded_like(randn(g, rows, n), t), padded_like(randn(g, rows, 2 * n, std=1.5), t)
    dx, dw = Padded(rows, k, t), torch.full((2 * n, k), float("nan"), device="cuda", dtype=grad_t)
    ws = torch.full((hip.gated_ffn_backward_workspace(rows, n, k) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    hip.op_gated_ffn_backward(dh, gu, x, wi, ws[:-64], act=act, dx=dx.t, dw=dw)
    torch.cuda.synchronize()
    dx.check()
    assert bool((ws[-64:] == 0xFF).all())
    gg, u, d = gu[:, :n].double(), gu[:, n:].double(), dh.double()
    a, slope = act64(gg, act)
    dz = torch.cat([d * u * slope, d * a], dim=1)
    off = (1 + gg.abs()) * ACT
    tdz = torch.cat([d.abs() * u.abs() * off, d.abs() * gg.abs() * off], dim=1) + dz.abs() * 2.0**-23
    (wx, tx), (ww, tw) = product_bounds(dz, tdz, wi.double(), x.double(), t, grad_t)
    close(dx.t, wx, tx, "dx")
    close(dw, ww, tw, "dw")


def test_gradients_of_no_rows_are_zero():
    x, dy = torch.empty(0, 64, device="cuda", dtype=BF16), torch.empty(0, 32, device="cuda", dtype=BF16)
    w, dw = torch.ones(32, 64, device="cuda", dtype=BF16), torch.full((32, 64), 5.0, device="cuda", dtype=BF16)
    db = torch.full((32,), 5.0, device="cuda")
    ws = torch.empty(max(1, hip.linear_backward_workspace(0, 32, 64, "gelu")), dtype=torch.uint8, device="cuda")
    hip.op_linear_backward(dy, x, w, ws, act="gelu", pre=dy, dx=torch.empty_like(x), dw=dw, dbias=db)
    dwi = torch.full((32, 64), 5.0, device="cuda")
    hip.op_gated_ffn_backward(dy[:, :16], dy, x, w, ws, dw=dwi)
    torch.cuda.synchronize()
    assert not bool(dw.any()) and not bool(db.any()) and not bool(dwi.any())


@pytest.mark.parametrize("t", [BF16, F16])
def test_one_row_whatever_its_stride(t):
    """One row's stride means nothing: a transposed column, whose row stride is 1, gives what a contiguous row gives."""
    n, k = 96, 200
    g = gen(31)
    w, norm_w = randn(g, n, k, std=0.1).to(t), 1 + randn(g, k, std=0.3)
    x, dy, dh, pre, dres = (randn(g, 1, c).to(t) for c in (k, n, n // 2, n, k))
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def run(row):
        def empty(c, dtype=t):
            return row(torch.full((1, c), 7.0, device="cuda").to(dtype))

        x_, dy_, dh_, pre_, dres_ = (row(v) for v in (x, dy, dh, pre, dres))
        out, kept, dx, h, gu, dxg = empty(n), empty(n), empty(k), empty(n // 2), empty(n), empty(k)
        y, s, ds, q = empty(k), empty(k), empty(k), empty(k, E4M3)
        dw, dwg, dnw = torch.empty_like(w), torch.empty(n, k, device="cuda"), torch.empty(k, device="cuda")
        db, scale, rstd = (torch.empty(c, device="cuda") for c in (n, 1, 1))
        hip.op_linear(x_, w, out, act="gelu", resid=dy_, pre=kept)
        hip.op_linear_backward(dy_, x_, w, ws, act="silu", pre=pre_, dx=dx, dw=dw, dbias=db)
        hip.op_gated_ffn(x_, w, h, gu=gu)
        hip.op_gated_ffn_backward(dh_, pre_, x_, w, ws, dx=dxg, dw=dwg)
        hip.op_rms_norm(x_, norm_w, EPS, y, resid=dres_, resid_out=s, rstd=rstd)
        hip.op_rms_norm_backward(dres_, s, norm_w, rstd, ds, dnw, ws, dres=x_)
        hip.op_quantize_rows(x_, q, scale)
        hip.op_linear(x_, w, dy_, resid=dy_.view(1, n))  # in place, by another view of the row
        torch.cuda.synchronize()
        return out, kept, dx, dw, db, h, gu, dxg, dwg, y, s, rstd, ds, dnw, q, scale, dy_

    for a, b in zip(run(lambda v: v.clone()), run(lambda v: v.clone().as_strided(v.shape, (1, 1)))):
        assert torch.equal(a.float(), b.float())


# ---------------------------------------------------------------- used together

class Block:
    """x + down(gated(norm(x + a))): one pre-norm feed-forward block and its gradients through the operators."""

    def __init__(self, rows, h, inter, t, seed):
        g = gen(seed)
        self.rows, self.h, self.inter, self.t = rows, h, inter, t
        self.a, self.resid = randn(g, rows, h).to(t), randn(g, rows, h)
        self.norm = 1 + randn(g, h, std=0.2)
        self.wi, self.wo = randn(g, 2 * inter, h, std=1 / math.sqrt(h)).to(t), randn(g, h, inter, std=1 / math.sqrt(inter)).to(t)
        self.dout = randn(g, rows, h)

        def e(*s, dtype=t):
            return torch.empty(*s, device="cuda", dtype=dtype)

        self.s, self.rstd, self.n, self.hid, self.gu, self.out = (e(rows, h, dtype=F32), e(rows, dtype=F32), e(rows, h),
                                                                  e(rows, inter), e(rows, 2 * inter), e(rows, h, dtype=F32))
        self.dhid, self.dn, self.ds = e(rows, inter), e(rows, h), e(rows, h, dtype=F32)
        self.dwi, self.dwo, self.dnorm = e(2 * inter, h, dtype=F32), e(h, inter, dtype=F32), e(h, dtype=F32)
        self.ws = e(max(hip.linear_backward_workspace(rows, h, inter, "none"), hip.gated_ffn_backward_workspace(rows, inter, h),
                        hip.rms_norm_backward_workspace(rows, h)), dtype=torch.uint8)

    def step(self, stream=None):
        hip.op_rms_norm(self.a, self.norm, EPS, self.n, resid=self.resid, resid_out=self.s, rstd=self.rstd, stream=stream)
        hip.op_gated_ffn(self.n, self.wi, self.hid, act="silu", gu=self.gu, stream=stream)
        hip.op_linear(self.hid, self.wo, self.out, resid=self.s, stream=stream)
        dy = self.dout.to(self.t)
        hip.op_linear_backward(dy, self.hid, self.wo, self.ws, dx=self.dhid, dw=self.dwo, stream=stream)
        hip.op_gated_ffn_backward(self.dhid, self.gu, self.n, self.wi, self.ws, act="silu", dx=self.dn, dw=self.dwi,
                                  stream=stream)
        hip.op_rms_norm_backward(self.dn, self.s, self.norm, self.rstd, self.ds, self.dnorm, self.ws, dres=self.dout,
                                 stream=stream)

    def outputs(self):
        return [self.s, self.out, self.ds, self.dwi, self.dwo, self.dnorm]


def test_block_gradients_against_autograd_and_differences():
    """The block in 64 bits on the same inputs: its output and gradients by autograd, and the loss's change along a
    random direction by differences.  The roundings to bf16 between the operators (n, h, gu, dy, dh, dgu, dn: relative
    2^-8 each at most, 2^-9 on average, independent) leave relative errors in norm of a few 2^-9; 2^-6 covers eight
    worst cases adding up in one direction by half."""
    b = Block(300, 256, 328, BF16, seed=1)
    b.step()
    torch.cuda.synchronize()

    def forward(a, resid, norm, wi, wo):
        s = a + resid
        n = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + EPS) * norm
        z = n @ wi.t()
        return s + (act64(z[:, :b.inter], "silu")[0] * z[:, b.inter:]) @ wo.t()

    leaves = [v.double().requires_grad_() for v in (b.a, b.resid, b.norm, b.wi, b.wo)]
    out = forward(*leaves)
    loss = (out * b.dout.double()).sum()
    loss.backward()
    got = [b.ds, b.ds, b.dnorm, b.dwi, b.dwo]
    assert float((b.out.double() - out.detach()).norm() / out.detach().norm()) < 2.0**-6
    for leaf, v, name in zip(leaves, got, ("a", "resid", "norm", "wi", "wo")):
        assert float((v.double() - leaf.grad).norm() / leaf.grad.norm()) < 2.0**-6, name
    g = gen(2)
    for leaf, v in zip(leaves, got):
        # the direction of the gradient itself with noise, so that the change does not cancel
        d = v.double() / v.double().norm() + torch.randn(leaf.shape, device="cuda", generator=g, dtype=torch.float64) * (
            0.1 / math.sqrt(leaf.numel()))
        step = 1e-4
        with torch.no_grad():
            up, down = ([p + (s * step * d if p is leaf else 0) for p in leaves] for s in (1, -1))
            change = ((forward(*up) - forward(*down)) * b.dout.double()).sum() / (2 * step)
        assert abs(float((v.double() * d).sum() / change) - 1) < 2.0**-6


def test_block_in_eight_bits():
    """norm -> e4m3 -> gated -> quantised -> linear + residual, against the same chain of the operators' definitions in
    64 bits on what each operator was given."""
    g = gen(4)
    rows, h, inter = 77, 512, 400
    a, resid, norm = randn(g, rows, h).to(BF16), randn(g, rows, h), 1 + randn(g, h, std=0.2)
    wi, wo = randn(g, 2 * inter, h, std=1 / math.sqrt(h)), randn(g, h, inter, std=1 / math.sqrt(inter))

    def e(*s, dtype=E4M3):
        return torch.empty(*s, device="cuda", dtype=dtype)

    qi, si, qo, so = e(2 * inter, h), e(2 * inter, dtype=F32), e(h, inter), e(h, dtype=F32)
    hip.op_quantize_rows(wi, qi, si)
    hip.op_quantize_rows(wo, qo, so)
    n8, ns, s = e(rows, h), e(rows, dtype=F32), e(rows, h, dtype=F32)
    hid, h8, hs, out = e(rows, inter, dtype=BF16), e(rows, inter), e(rows, dtype=F32), e(rows, h, dtype=F32)
    hip.op_rms_norm(a, norm, EPS, n8, resid=resid, resid_out=s, scales=ns)
    hip.op_gated_ffn(n8, qi, hid, act="gelu", x_scale=ns, w_scale=si)
    hip.op_quantize_rows(hid, h8, hs)
    hip.op_linear(h8, qo, out, resid=s, x_scale=hs, w_scale=so)
    torch.cuda.synchronize()
    z = (n8.double() * ns.double()[:, None]) @ (qi.double() * si.double()[:, None]).t()
    want = act64(z[:, :inter], "gelu")[0] * z[:, inter:]
    assert float((hid.double() - want).norm() / want.norm()) < 2.0**-8
    want = s.double() + (h8.double() * hs.double()[:, None]) @ (qo.double() * so.double()[:, None]).t()
    assert float((out.double() - want).norm() / want.norm()) < 1e-5
    # and the whole chain is the unquantised block's to the precision of 8 bits (each of four operands off by at most
    # 2^-4, about 2^-5.5 on average)
    s64 = a.double() + resid.double()
    n = s64 / torch.sqrt((s64 * s64).mean(dim=1, keepdim=True) + EPS) * norm.double()
    z = n @ wi.double().t()
    want = (act64(z[:, :inter], "gelu")[0] * z[:, inter:]) @ wo.double().t()
    assert float((out.double() - s64 - want).norm() / want.norm()) < 4 * 2.0**-4


def test_block_on_another_stream_and_in_a_graph():
    """The block on a stream of its own, then captured: every replay has the eager run's bits, with eager work on other
    inputs between the replays.  Two graphs that share one workspace run one after the other on one stream."""
    b, other = Block(130, 256, 264, BF16, seed=5), Block(130, 256, 264, BF16, seed=6)
    b.step()
    other.step()
    torch.cuda.synchronize()
    want, want2 = [t.clone() for t in b.outputs()], [t.clone() for t in other.outputs()]
    st = torch.cuda.Stream()
    for t in b.outputs():
        t.zero_()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b.step(stream=st.cuda_stream)
    st.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(b.outputs(), want))
    other.ws = b.ws
    graphs = []
    for blk in (b, other):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            blk.step(stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(gr)
    for _ in range(3):
        for t in b.outputs() + other.outputs():
            t.fill_(3.0)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(b.outputs(), want))
        assert all(torch.equal(x, y) for x, y in zip(other.outputs(), want2))
        Block(64, 128, 72, F16, seed=7).step()
        torch.cuda.synchronize()


def test_blocks_on_two_streams_at_once():
    """Two blocks with workspaces of their own, on two streams without order between them."""
    a, b = Block(700, 512, 520, BF16, seed=8), Block(700, 512, 520, BF16, seed=9)
    a.step()
    b.step()
    torch.cuda.synchronize()
    want = [t.clone() for t in a.outputs() + b.outputs()]
    for t in a.outputs() + b.outputs():
        t.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for blk, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                blk.step(stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a.outputs() + b.outputs(), want))


# ---------------------------------------------------------------- far offsets

def roomy(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def some(rows):
    """Row indices on both sides of 2^31 elements, the first and the last."""
    return torch.tensor([0, 1, rows // 2, rows - 4000, rows - 2, rows - 1], device="cuda")


def test_rows_past_2_31_elements_norms():
    roomy(40)
    rows, h = 140000, 16384
    g = gen(11)
    x = torch.empty(rows, h, device="cuda", dtype=BF16)
    for i in range(0, rows, 20000):
        x[i:i + 20000] = randn(g, 20000, h)[: rows - i]
    w, out, q, scales = 1 + randn(g, h, std=0.2), torch.empty_like(x), torch.empty(rows, h, device="cuda", dtype=E4M3), \
        torch.empty(rows, device="cuda")
    rstd = torch.empty(rows, device="cuda")
    hip.op_rms_norm(x, w, EPS, out, rstd=rstd)
    hip.op_quantize_rows(x, q, scales)
    torch.cuda.synchronize()
    i = some(rows)
    v = x[i].double()
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * w.double()
    close(out[i], y, y.abs() * (half(BF16) + (h + 32) * 2.0**-24), "out")
    assert torch.equal(q[i].double(), nearest_e4m3(v * 448 / v.abs().amax(dim=1, keepdim=True)))
    hip.op_rms_norm_backward(x, x, w, rstd, out)
    torch.cuda.synchronize()
    r = rstd[i].double()[:, None]
    n, gy = v * r, v * w.double()
    want = r * (gy - n * (gy * n).mean(dim=1, keepdim=True))
    size = (gy * n).abs().mean(dim=1, keepdim=True)
    close(out[i], want, r * (gy.abs() * 8 + n.abs() * size * (h + 16)) * 2.0**-24 + want.abs() * half(BF16), "ds")


def test_more_rows_than_a_launch_has_along_x():
    """2^32 threads and more: rows that repeat those of a small call get its bits."""
    roomy(12)
    base, h, rows = 4099, 8, 2**26 + 9
    g = gen(13)
    few, w = randn(g, base, h).to(BF16), 1 + randn(g, h, std=0.2)
    x = few.repeat(rows // base + 1, 1)[:rows]

    def run(x):
        out, q = torch.empty_like(x), torch.empty(x.shape, device="cuda", dtype=E4M3)
        scales, rstd = (torch.empty(x.shape[0], device="cuda") for _ in range(2))
        hip.op_rms_norm(x, w, EPS, out, rstd=rstd)
        hip.op_quantize_rows(x, q, scales)
        torch.cuda.synchronize()
        return out.view(torch.int16), q.view(torch.uint8), scales[:, None], rstd[:, None]

    for all_rows, want in zip(run(x), run(few)):
        whole = rows // base * base
        assert bool((all_rows[:whole].view(-1, base, want.shape[1]) == want).all())
        assert torch.equal(all_rows[whole:], want[:rows - whole])


def test_rows_past_2_31_elements_products():
    roomy(60)
    rows, n, k = 70000, 32768, 64
    g = gen(12)
    x, w = randn(g, rows, k).to(BF16), randn(g, n, k, std=0.125).to(BF16)
    out, pre = torch.empty(rows, n, device="cuda", dtype=BF16), torch.empty(rows, n, device="cuda", dtype=BF16)
    hip.op_linear(x, w, out, act="relu", pre=pre)
    torch.cuda.synchronize()
    i = some(rows)
    z = x[i].double() @ w.double().t()
    tol = z.abs() * half(BF16) + (x[i].double().abs() @ w.double().abs().t()) * (k + 4) * 2.0**-23
    close(pre[i], z, tol, "pre")
    close(out[i], z.clamp_min(0), tol, "out")
    # gradients: dy = out, a pre-activation that the relu passes on every other column
    dx, dw = torch.empty_like(x), torch.empty(n, k, device="cuda")
    ws = torch.empty(hip.linear_backward_workspace(rows, n, k, "relu"), dtype=torch.uint8, device="cuda")
    hip.op_linear_backward(out, x, w, ws, act="relu", pre=pre, dx=dx, dw=dw)
    torch.cuda.synchronize()
    dz = out[i].double() * (pre[i] > 0)
    want = dz @ w.double()
    close(dx[i], want, want.abs() * half(BF16) + (dz.abs() @ w.double().abs()) * (n + 4) * 2.0**-23, "dx")
    c = torch.tensor([0, 5, n // 2, n - 1], device="cuda")
    dz = out[:, c].double() * (pre[:, c] > 0)
    want = dz.t() @ x.double()
    close(dw[c], want, (dz.abs().t() @ x.double().abs()) * (rows + 32) * 2.0**-23 + want.abs() * half(F32), "dw")
    del out, pre, ws
    inter = n // 2
    h, gu = torch.empty(rows, inter, device="cuda", dtype=BF16), torch.empty(rows, n, device="cuda", dtype=BF16)
    hip.op_gated_ffn(x, w, h, act="relu", gu=gu)
    torch.cuda.synchronize()
    close(gu[i], z, tol, "gu")
    ws = torch.empty(hip.gated_ffn_backward_workspace(rows, inter, k), dtype=torch.uint8, device="cuda")
    hip.op_gated_ffn_backward(h, gu, x, w, ws, act="relu", dx=dx)
    torch.cuda.synchronize()
    a, u, d = gu[i, :inter].double().clamp_min(0), gu[i, inter:].double(), h[i].double()
    dz = torch.cat([d * u * (gu[i, :inter] > 0), d * a], dim=1)
    want = dz @ w.double()
    close(dx[i], want, want.abs() * half(BF16) + (dz.abs() @ w.double().abs()) * (half(BF16) * 1.01 + (n + 4) * 2.0**-23), "dx")
