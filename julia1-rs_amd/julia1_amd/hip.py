"""ctypes binding of libjulia1_hip.so (include/julia1_hip.h, include/julia1_hip_ops.h).

The library must have been built (julia1-rs_amd/build.py or
__graft_entry__.build()); loading fails loudly otherwise — there is no
fallback path.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

from . import abi

_lib = None

EXPORTS = (
    "jh_create", "jh_forward", "jh_forward_padded", "jh_stage", "jh_execute", "jh_scores", "jh_stream", "jh_submit",
    "jh_collect",
    "jh_set_graph", "jh_set_splitk", "jh_name", "jh_destroy", "jh_last_error", "jh_rope_table", "jh_debug_tokens",
    "jh_debug_encode", "jh_debug_workspace_limit", "jh_profile", "jh_profile_read", "jh_profile_replay",
    "jh_op_gemm", "jh_op_gemm_splitk", "jh_op_gemm_splitk_noalloc", "jh_op_gemm_ln", "jh_op_gemm_ws", "jh_op_pack_ws",
    "jh_op_interleave_geglu",
    "jh_op_embed_ln", "jh_op_layer_norm", "jh_op_final_norm",
    "jh_op_gather_f32", "jh_op_scorer", "jh_op_attention", "jh_op_attention_wide", "jh_op_attention_unsplit",
    "jh_op_rms_norm", "jh_op_rms_norm_backward", "jh_op_rms_norm_backward_workspace", "jh_op_quantize_rows",
    "jh_op_linear", "jh_op_linear_backward", "jh_op_linear_backward_workspace", "jh_op_linear_plan",
    "jh_op_gated_ffn", "jh_op_gated_ffn_backward", "jh_op_gated_ffn_backward_workspace",
)


class KernelStat(C.Structure):
    _fields_ = [("name", C.c_char_p), ("launches", C.c_uint32), ("ms", C.c_double), ("flops", C.c_double),
                ("bytes", C.c_double)]


class LinearLaunch(C.Structure):
    _fields_ = [("kernel", C.c_int), ("parts", C.c_int), ("rows", C.c_size_t)]


class HipError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"[{code}] {msg}")
        self.code = code


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(abi.LIB_PATH):
            raise RuntimeError(f"{abi.LIB_PATH} is not built; run julia1-rs_amd/build.py")
        L = C.CDLL(abi.LIB_PATH)
        vp, sz, u32 = C.c_void_p, C.c_size_t, C.c_uint32
        L.jh_create.argtypes = [vp, vp, C.c_int, C.POINTER(vp)]
        L.jh_forward.argtypes = [vp, vp, sz, vp, vp, vp, sz, vp, sz, vp]
        L.jh_forward_padded.argtypes = [vp, vp, sz, sz, vp, vp, vp, vp, vp]
        L.jh_stage.argtypes = [vp, vp, sz, vp, vp, vp, sz, vp, sz]
        L.jh_execute.argtypes = [vp]
        L.jh_scores.argtypes = [vp, vp, sz]
        L.jh_submit.argtypes = [vp, vp, sz, vp, vp, vp, sz, vp, sz, C.POINTER(C.c_uint64)]
        L.jh_collect.argtypes = [vp, C.c_uint64, vp, sz]
        L.jh_stream.argtypes = [vp]
        L.jh_stream.restype = vp
        L.jh_set_graph.argtypes = [vp, C.c_int]
        L.jh_set_splitk.argtypes = [vp, C.c_int]
        L.jh_name.argtypes = [vp]
        L.jh_name.restype = C.c_char_p
        L.jh_destroy.argtypes = [vp]
        L.jh_destroy.restype = None
        L.jh_last_error.argtypes = []
        L.jh_last_error.restype = C.c_char_p
        L.jh_rope_table.argtypes = [C.c_float, u32, u32, vp, vp]
        L.jh_rope_table.restype = None
        L.jh_debug_tokens.argtypes = [vp, vp, vp, sz]
        L.jh_debug_encode.argtypes = [vp, u32, vp, sz]
        L.jh_debug_workspace_limit.argtypes = [vp, sz]
        L.jh_profile.argtypes = [vp, C.c_int]
        L.jh_profile_read.argtypes = [vp, vp, sz, C.POINTER(sz)]
        L.jh_profile_replay.argtypes = [vp, C.c_char_p, sz, C.POINTER(C.c_double)]
        L.jh_op_gemm.argtypes = [C.c_int, vp, sz, vp, sz, vp, sz, sz, vp, sz, sz, vp, vp, vp, vp, sz, vp]
        L.jh_op_gemm_splitk.argtypes = [C.c_int, vp, sz, vp, sz, vp, sz, sz, vp, sz, sz, vp, vp, vp, vp, sz, vp, sz,
                                        C.c_int, vp]
        L.jh_op_gemm_splitk_noalloc.argtypes = [C.c_int, vp, sz, vp, sz, vp, sz, sz, vp, sz, sz, vp, vp, vp, vp,
                                                sz, C.c_int, vp]
        L.jh_op_gemm_ln.argtypes = [C.c_int, vp, sz, sz, vp, sz, sz, vp, sz, sz, vp, vp, vp, sz, vp, vp, C.c_float,
                                    vp]
        L.jh_op_gemm_ws.argtypes = [C.c_int, vp, sz, sz, vp, sz, sz, vp, sz, sz, vp, vp, vp, vp, sz, vp]
        L.jh_op_pack_ws.argtypes = [vp, sz, sz, vp]
        L.jh_op_interleave_geglu.argtypes = [vp, sz, sz, vp]
        L.jh_op_interleave_geglu.restype = None
        L.jh_op_embed_ln.argtypes = [vp, sz, vp, vp, C.c_float, sz, vp, vp, vp]
        L.jh_op_layer_norm.argtypes = [vp, sz, vp, vp, C.c_float, sz, vp, vp]
        L.jh_op_final_norm.argtypes = [vp, sz, vp, vp, vp, vp, vp, C.c_float, sz, vp, vp]
        L.jh_op_gather_f32.argtypes = [vp, vp, sz, sz, vp, vp]
        L.jh_op_scorer.argtypes = [vp, sz, sz, vp, C.c_float, vp, vp]
        L.jh_op_attention.argtypes = [vp, sz, vp, vp, sz, vp, sz, vp, sz, sz, C.c_int, C.c_float, vp]
        L.jh_op_attention_wide.argtypes = L.jh_op_attention.argtypes
        L.jh_op_attention_unsplit.argtypes = L.jh_op_attention.argtypes[:-1] + [C.c_int, vp]
        i32, f32 = C.c_int, C.c_float
        L.jh_op_rms_norm.argtypes = [i32, vp, sz, i32, vp, sz, vp, sz, sz, sz, vp, f32, i32, vp, sz, vp, vp, vp]
        L.jh_op_rms_norm_backward.argtypes = [i32, vp, sz, i32, vp, sz, sz, sz, vp, vp, i32, vp, sz, vp, sz, vp, vp, sz,
                                              vp]
        L.jh_op_quantize_rows.argtypes = [i32, vp, sz, sz, sz, vp, sz, vp, vp]
        L.jh_op_linear.argtypes = [i32, vp, sz, vp, sz, vp, vp, sz, sz, vp, i32, vp, sz, i32, vp, sz, vp, sz, vp]
        L.jh_op_linear_backward.argtypes = [i32, vp, sz, vp, sz, sz, vp, sz, sz, i32, vp, sz, vp, sz, i32, vp, vp, vp,
                                            sz, vp]
        L.jh_op_gated_ffn.argtypes = [i32, vp, sz, vp, sz, vp, vp, sz, sz, i32, vp, sz, vp, sz, vp]
        L.jh_op_gated_ffn_backward.argtypes = [i32, vp, sz, vp, sz, vp, sz, sz, vp, sz, sz, i32, vp, sz, i32, vp, vp,
                                               sz, vp]
        L.jh_op_linear_plan.argtypes = [i32, i32, i32, sz, sz, sz, C.POINTER(LinearLaunch)]
        L.jh_op_rms_norm_backward_workspace.argtypes = [sz, sz]
        L.jh_op_linear_backward_workspace.argtypes = [sz, sz, sz, i32]
        L.jh_op_gated_ffn_backward_workspace.argtypes = [sz, sz, sz]
        for name in ("rms_norm", "linear", "gated_ffn"):
            getattr(L, f"jh_op_{name}_backward_workspace").restype = sz
        _lib = L
    return _lib


def check(rc):
    if rc != 0:
        raise HipError(rc, lib().jh_last_error().decode())


def _p(a):
    return None if a is None else a.ctypes.data


def rope_table(theta: float, positions: int, head_dim: int = 64):
    half = head_dim // 2
    c = np.zeros((positions, half), dtype=np.float32)
    s = np.zeros((positions, half), dtype=np.float32)
    lib().jh_rope_table(theta, head_dim, positions, _p(c), _p(s))
    return c, s


class HipModel:
    """The `Backend::Hip` model: jh_create / jh_forward / jh_name / jh_destroy."""

    def __init__(self, weight_set, ordinal: int = 0):
        self._ws = weight_set
        h = C.c_void_p()
        check(lib().jh_create(C.addressof(weight_set.config), C.addressof(weight_set.weights), ordinal, C.byref(h)))
        self.h = h
        self.cfg = weight_set.cfg

    @property
    def name(self) -> str:
        return lib().jh_name(self.h).decode()

    def forward(self, b) -> np.ndarray:
        scores = np.zeros(b.marker_rows.size, dtype=np.float32)
        check(lib().jh_forward(self.h, _p(b.ids), b.tokens, _p(b.starts), _p(b.lens), _p(b.qtypes), b.lens.size,
                               _p(b.marker_rows), b.marker_rows.size, _p(scores)))
        return scores

    def forward_padded(self, ids, lens, qtypes, markers, marker_starts) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        B, L = ids.shape
        lens = np.ascontiguousarray(lens, dtype=np.uint32)
        qtypes = np.ascontiguousarray(qtypes, dtype=np.uint8)
        markers = np.ascontiguousarray(markers, dtype=np.uint32)
        marker_starts = np.ascontiguousarray(marker_starts, dtype=np.uint32)
        scores = np.zeros(int(marker_starts[-1]) if B else 0, dtype=np.float32)
        check(lib().jh_forward_padded(self.h, _p(ids), B, L, _p(lens), _p(qtypes), _p(markers), _p(marker_starts),
                                      _p(scores)))
        return scores

    def submit(self, b) -> int:
        """jh_submit: enqueue a forward without waiting; returns its ticket."""
        t = C.c_uint64(0)
        check(lib().jh_submit(self.h, _p(b.ids), b.tokens, _p(b.starts), _p(b.lens), _p(b.qtypes), b.lens.size,
                              _p(b.marker_rows), b.marker_rows.size, C.byref(t)))
        return t.value

    def collect(self, ticket: int, m: int) -> np.ndarray:
        """jh_collect: wait for a submitted forward and return its m scores."""
        out = np.zeros(m, dtype=np.float32)
        check(lib().jh_collect(self.h, ticket, _p(out), m))
        return out

    def stage(self, b):
        self._staged = b
        check(lib().jh_stage(self.h, _p(b.ids), b.tokens, _p(b.starts), _p(b.lens), _p(b.qtypes), b.lens.size,
                             _p(b.marker_rows), b.marker_rows.size))

    def execute(self):
        check(lib().jh_execute(self.h))

    def scores(self, m: int) -> np.ndarray:
        out = np.zeros(m, dtype=np.float32)
        check(lib().jh_scores(self.h, _p(out), m))
        return out

    def set_graph(self, on: bool):
        check(lib().jh_set_graph(self.h, 1 if on else 0))

    def set_splitk(self, on: bool):
        check(lib().jh_set_splitk(self.h, 1 if on else 0))

    @property
    def stream(self) -> int:
        return lib().jh_stream(self.h) or 0

    def debug_tokens(self, t: int):
        ids = np.zeros(t, dtype=np.uint32)
        pos = np.zeros(t, dtype=np.uint32)
        check(lib().jh_debug_tokens(self.h, _p(ids), _p(pos), t))
        return ids, pos

    def debug_encode(self, t: int, layers: int) -> np.ndarray:
        x = np.zeros((t, self.cfg.hidden), dtype=np.float32)
        check(lib().jh_debug_encode(self.h, layers, _p(x), t))
        return x

    def debug_workspace_limit(self, nbytes: int):
        """jh_debug_workspace_limit: later workspace growths past `nbytes` fail with JH_ERR_ALLOC (0 = off)."""
        check(lib().jh_debug_workspace_limit(self.h, nbytes))

    def profile(self, on: bool):
        check(lib().jh_profile(self.h, 1 if on else 0))

    def profile_read(self) -> list:
        """[{name, launches, ms, flops, bytes}] summed since the last read (device time from HIP events)."""
        arr = (KernelStat * 32)()
        n = C.c_size_t()
        check(lib().jh_profile_read(self.h, arr, 32, C.byref(n)))
        return [dict(name=arr[i].name.decode(), launches=arr[i].launches, ms=arr[i].ms, flops=arr[i].flops,
                     bytes=arr[i].bytes) for i in range(n.value)]

    def profile_replay(self, kernel_class: str, reps: int = 50) -> float:
        """Mean device µs of one launch of a GEMM/attention class, replayed back to back
        (see jh_profile_replay); valid right after a profiled forward."""
        us = C.c_double()
        check(lib().jh_profile_replay(self.h, kernel_class.encode(), reps, C.byref(us)))
        return us.value

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.jh_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


# ---------------------------------------------------------------- op level (device tensors via torch)

def _dp(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def op_gemm(epi, x, w, out, rows=None, gather=None, col=0, bias=None, pos=None, cos=None, sin=None, rope_cols=0,
            stream=None):
    """x, w bf16 torch tensors (2-D), out torch tensor; see jh_op_gemm."""
    rows = x.shape[0] if rows is None else rows
    n, k = w.shape
    check(lib().jh_op_gemm(epi, _dp(x), x.stride(0), _dp(gather), rows, _dp(w), n, k, _dp(out), out.stride(0), col,
                           _dp(bias), _dp(pos), _dp(cos), _dp(sin), rope_cols, stream))


def op_gemm_splitk(epi, x, w, out, workspace, splits=0, rows=None, gather=None, col=0, bias=None, pos=None, cos=None,
                   sin=None, rope_cols=0, stream=None):
    """jh_op_gemm_splitk: like op_gemm with a torch workspace tensor for the FP32 partials."""
    rows = x.shape[0] if rows is None else rows
    n, k = w.shape
    check(lib().jh_op_gemm_splitk(epi, _dp(x), x.stride(0), _dp(gather), rows, _dp(w), n, k, _dp(out), out.stride(0),
                                  col, _dp(bias), _dp(pos), _dp(cos), _dp(sin), rope_cols, _dp(workspace),
                                  workspace.numel() * workspace.element_size(), splits, stream))


def op_gemm_ln(epi, xf, w, out, ln_w, ln_b=None, eps=1e-5, rows=None, col=0, pos=None, cos=None, sin=None,
               rope_cols=0, stream=None):
    """jh_op_gemm_ln: X = bf16(LayerNorm(xf)) computed inside the GEMM; xf an FP32 torch tensor (2-D)."""
    rows = xf.shape[0] if rows is None else rows
    n, k = w.shape
    check(lib().jh_op_gemm_ln(epi, _dp(xf), xf.stride(0), rows, _dp(w), n, k, _dp(out), out.stride(0), col,
                              _dp(pos), _dp(cos), _dp(sin), rope_cols, _dp(ln_w), _dp(ln_b), eps, stream))


def op_gemm_splitk_noalloc(epi, x, w, out, splits=0, rows=None, gather=None, col=0, bias=None, pos=None, cos=None,
                           sin=None, rope_cols=0, stream=None):
    """jh_op_gemm_splitk_noalloc: op_gemm_splitk with the library's fixed scratch instead of a workspace."""
    rows = x.shape[0] if rows is None else rows
    n, k = w.shape
    check(lib().jh_op_gemm_splitk_noalloc(epi, _dp(x), x.stride(0), _dp(gather), rows, _dp(w), n, k, _dp(out),
                                          out.stride(0), col, _dp(bias), _dp(pos), _dp(cos), _dp(sin), rope_cols,
                                          splits, stream))


def pack_ws(w):
    """bf16 torch tensor [n, k] (PyTorch Linear layout; the GEGLU interleave for Wi) -> the same values on the
    device in the weight-stationary kernel's fragment order (jh_op_pack_ws)."""
    import torch
    src = w.detach().to("cpu").contiguous().view(torch.int16).numpy()
    n, k = src.shape
    dst = np.empty_like(src)
    check(lib().jh_op_pack_ws(src.ctypes.data_as(C.c_void_p), n, k, dst.ctypes.data_as(C.c_void_p)))
    return torch.from_numpy(dst).view(torch.bfloat16).cuda()


def op_gemm_ws(epi, x, w_packed, n, k, out, rows=None, col=0, bias=None, pos=None, cos=None, sin=None, rope_cols=0,
               stream=None):
    """jh_op_gemm_ws: the weight-stationary GEMM on W packed by pack_ws (K = 768 with N % 256 == 0, or K = 1152
    with N % 128 == 0 and the residual epilogue)."""
    rows = x.shape[0] if rows is None else rows
    check(lib().jh_op_gemm_ws(epi, _dp(x), x.stride(0), rows, _dp(w_packed), n, k, _dp(out), out.stride(0), col,
                              _dp(bias), _dp(pos), _dp(cos), _dp(sin), rope_cols, stream))


def interleave_geglu(wi: np.ndarray) -> np.ndarray:
    wi = np.ascontiguousarray(wi, dtype=np.float32)
    out = np.empty_like(wi)
    lib().jh_op_interleave_geglu(_p(wi), wi.shape[0] // 2, wi.shape[1], _p(out))
    return out


def op_embed_ln(ids, table, w, eps, x, xn, stream=None):
    check(lib().jh_op_embed_ln(_dp(ids), ids.numel(), _dp(table), _dp(w), eps, table.shape[1], _dp(x), _dp(xn), stream))


def op_layer_norm(x, w, b, eps, out, stream=None):
    check(lib().jh_op_layer_norm(_dp(x), x.shape[0], _dp(w), _dp(b), eps, x.shape[1], _dp(out), stream))


def op_final_norm(x, fw, type_emb, tok_meta, hw, hb, eps, out, stream=None):
    check(lib().jh_op_final_norm(_dp(x), x.shape[0], _dp(fw), _dp(type_emb), _dp(tok_meta), _dp(hw), _dp(hb), eps,
                                 x.shape[1], _dp(out), stream))


def op_gather_f32(src, idx, dst, stream=None):
    check(lib().jh_op_gather_f32(_dp(src), _dp(idx), idx.numel(), src.shape[1], _dp(dst), stream))


def op_scorer(z, w2, b2, out, stream=None):
    check(lib().jh_op_scorer(_dp(z), z.shape[0], z.shape[1], _dp(w2), b2, _dp(out), stream))


def op_attention(q, ldq, k, v, ldkv, out, ldo, tiles, heads, window, scale=0.125, stream=None, wide=False,
                 key_split=True):
    """q/k/v/out torch bf16 tensors (base pointers of the first row/col); tiles torch int32 [n, 5] of at most
    128 queries each, or 256 with wide=True (eight-wave work items, jh_op_attention_wide); key_split=False keeps
    each query's keys in one wave (jh_op_attention_unsplit)."""
    if not key_split:
        check(lib().jh_op_attention_unsplit(_dp(q), ldq, _dp(k), _dp(v), ldkv, _dp(out), ldo, _dp(tiles), tiles.shape[0],
                                            heads, window, scale, 1 if wide else 0, stream))
        return
    fn = lib().jh_op_attention_wide if wide else lib().jh_op_attention
    check(fn(_dp(q), ldq, _dp(k), _dp(v), ldkv, _dp(out), ldo, _dp(tiles), tiles.shape[0], heads, window, scale,
             stream))


# ---------------------------------------------------------------- RMS norm, linear layers, gated projections

ACTS = {"none": abi.ACT_NONE, "relu": abi.ACT_RELU, "gelu": abi.ACT_GELU, "gelu_tanh": abi.ACT_GELU_TANH,
        "silu": abi.ACT_SILU}
_TYPES = {}


def _invalid(msg):
    raise HipError(abi.JH_ERR_INVALID, msg)


def _dtype_codes():
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16,
                       torch.float8_e4m3fn: abi.E4M3})
    return _TYPES


def _type(t):
    """The element type code of a torch tensor."""
    code = _TYPES.get(t.dtype)
    if code is None:
        code = _dtype_codes().get(t.dtype)
        if code is None:
            _invalid(f"no such element type: {t.dtype}")
    return code


# These run before every launch of a few microseconds, so they ask a tensor for no more than they need.

def _first(name, t):
    """(address, row stride, shape, device) of an operator's first operand, a 2-D tensor on the current device (where
    the kernels are launched)."""
    shape = t.shape
    if len(shape) != 2:
        _invalid(f"{name}: needs a matrix")
    ld, one = t.stride()
    if one != 1 and shape[1] > 1:
        _invalid(f"{name}: needs contiguous rows")
    dev = t.get_device()
    if dev < 0 or dev != _current_device():
        _invalid(f"{name}: on {t.device}, which is not the current device")
    return t.data_ptr(), ld, shape, dev


def _current_device():
    global _current_device
    import torch
    _current_device = torch.cuda.current_device
    return _current_device()


def _mat(name, t, shape, dev, dtype):
    """(address, row stride) of a 2-D tensor of the wanted shape, type and device; (None, 0) for None."""
    if t is None:
        return None, 0
    if t.shape == shape and t.dtype is dtype and t.get_device() == dev:
        ld, one = t.stride()
        if one == 1 or shape[1] <= 1:
            return t.data_ptr(), ld
        _invalid(f"{name}: needs contiguous rows")
    _invalid(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, expected {dtype} {tuple(shape)} on the first operand's "
             "device")


def _weight(name, t, shape, dev, dtype):
    """Address of a contiguous matrix; None for None."""
    if t is None:
        return None
    if t.shape == shape and t.dtype is dtype and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _invalid(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, expected contiguous {dtype} {tuple(shape)} on the first "
             "operand's device")


def _vec(name, t, n, dev):
    """Address of a contiguous f32 vector of n values; None for None."""
    if t is None:
        return None
    if t.numel() == n and _type(t) == abi.F32 and t.is_contiguous() and t.get_device() == dev:
        return t.data_ptr()
    _invalid(f"{name}: needs {n} contiguous float32 values on the first operand's device")


def _space(t, dev):
    if t is None:
        return None, 0
    if not t.is_contiguous() or t.get_device() != dev:
        _invalid("workspace: needs contiguous memory on the first operand's device")
    return t.data_ptr(), t.numel() * t.element_size()


def _act(name):
    code = ACTS.get(name)
    if code is None:
        _invalid(f"unknown activation {name!r}")
    return code


def _bytes(n):
    if lib().jh_last_error():
        raise HipError(abi.JH_ERR_INVALID, lib().jh_last_error().decode())
    return n


def op_rms_norm(x, w, eps, out, resid=None, resid_out=None, scales=None, rstd=None, stream=None):
    """jh_op_rms_norm: out = RMS norm of s = x + resid, times w; s goes to resid_out (which may be resid).  out of
    torch.float8_e4m3fn takes e4m3 codes and scales their f32 scale per row; rstd (f32) is kept for the backward."""
    xp, ldx, shape, dev = _first("x", x)
    rows, h = shape
    op, ldo = _mat("out", out, shape, dev, out.dtype)
    rp = sp = cp = tp = None
    rt = ldr = lds = 0
    if scales is not None:
        cp = _vec("scales", scales, rows, dev)
    if rstd is not None:
        tp = _vec("rstd", rstd, rows, dev)
    if resid is not None or resid_out is not None:
        dt = (resid_out if resid is None else resid).dtype
        rt = _type(resid_out if resid is None else resid)
        rp, ldr = _mat("resid", resid, shape, dev, dt)
        sp, lds = _mat("resid_out", resid_out, shape, dev, dt)
    check(lib().jh_op_rms_norm(_type(x), xp, ldx, rt, rp, ldr, sp, lds, rows, h, _vec("w", w, h, dev), eps, _type(out),
                               op, ldo, cp, tp, stream))


def op_rms_norm_backward(dy, s, w, rstd, ds, dw=None, workspace=None, dres=None, stream=None):
    """jh_op_rms_norm_backward: ds (+ dres) and dw from dy, with s = resid_out (or x) and rstd of op_rms_norm; dw
    needs a workspace tensor of rms_norm_backward_workspace(rows, hidden) bytes."""
    yp, ldy, shape, dev = _first("dy", dy)
    rows, h = shape
    (sp, lds), (dp, ldd) = _mat("s", s, shape, dev, s.dtype), _mat("ds", ds, shape, dev, ds.dtype)
    rp, ldr = _mat("dres", dres, shape, dev, ds.dtype)
    wp, wb = _space(workspace, dev)
    check(lib().jh_op_rms_norm_backward(_type(dy), yp, ldy, _type(s), sp, lds, rows, h, _vec("w", w, h, dev),
                                        _vec("rstd", rstd, rows, dev), _type(ds), rp, ldr, dp, ldd,
                                        _vec("dw", dw, h, dev), wp, wb, stream))


def rms_norm_backward_workspace(rows, hidden) -> int:
    return _bytes(lib().jh_op_rms_norm_backward_workspace(rows, hidden))


def op_quantize_rows(x, q, scales, stream=None):
    """jh_op_quantize_rows: e4m3 codes q (torch.float8_e4m3fn) of x's rows and their f32 scales."""
    xp, ldx, shape, dev = _first("x", x)
    rows, n = shape
    qp, ldq = _mat("q", q, shape, dev, q.dtype)
    if _type(q) != abi.E4M3:
        _invalid("q: needs torch.float8_e4m3fn")
    check(lib().jh_op_quantize_rows(_type(x), xp, ldx, rows, n, qp, ldq, _vec("scales", scales, rows, dev), stream))


def op_linear(x, w, out, bias=None, act="none", resid=None, x_scale=None, w_scale=None, pre=None, stream=None):
    """jh_op_linear: out = act(x w^T + bias) + resid; x and w of one type (bf16, f16, or float8_e4m3fn with x_scale and
    w_scale), out f32 or their type (bf16 for e4m3); resid may be out; pre keeps x w^T + bias for the backward."""
    xp, ldx, (rows, k), dev = _first("x", x)
    n, dt, ot = w.shape[0], x.dtype, out.dtype
    shape = (rows, n)
    op, ldo = _mat("out", out, shape, dev, ot)
    rp = pp = xs = ws = bp = None
    ldr = ldp = 0
    if resid is not None:
        rp, ldr = _mat("resid", resid, shape, dev, ot)
    if pre is not None:
        pp, ldp = _mat("pre", pre, shape, dev, dt)
    if x_scale is not None:
        xs = _vec("x_scale", x_scale, rows, dev)
    if w_scale is not None:
        ws = _vec("w_scale", w_scale, n, dev)
    if bias is not None:
        bp = _vec("bias", bias, n, dev)
    check(lib().jh_op_linear(_type(x), xp, ldx, xs, rows, _weight("w", w, (n, k), dev, dt), ws, n, k, bp, _act(act), rp,
                             ldr, _type(out), op, ldo, pp, ldp, stream))


def op_linear_backward(dy, x, w, workspace, act="none", pre=None, dx=None, dw=None, dbias=None, stream=None):
    """jh_op_linear_backward: whichever of dx, dw (f32 or x's type) and dbias (f32) are given, from dy and (act not
    "none") pre; workspace of linear_backward_workspace(rows, n, k, act) bytes."""
    yp, ldy, shape, dev = _first("dy", dy)
    rows, n = shape
    k, dt = w.shape[1], dy.dtype
    (xp, ldx), (dp, ldd) = _mat("x", x, (rows, k), dev, dt), _mat("dx", dx, (rows, k), dev, dt)
    pp, ldp = _mat("pre", pre, shape, dev, dt)
    wp, wb = _space(workspace, dev)
    check(lib().jh_op_linear_backward(_type(dy), yp, ldy, xp, ldx, rows, _weight("w", w, (n, k), dev, dt), n, k,
                                      _act(act), pp, ldp, dp, ldd, _type(dy if dw is None else dw),
                                      _weight("dw", dw, (n, k), dev, dt if dw is None else dw.dtype),
                                      _vec("dbias", dbias, n, dev), wp, wb, stream))


def linear_backward_workspace(rows, n, k, act="none") -> int:
    return _bytes(lib().jh_op_linear_backward_workspace(rows, n, k, _act(act)))


def linear_plan(product, dtype, rows, n, k, out_dtype=None):
    """jh_op_linear_plan: [(kernel, parts, rows)] of the one or two launches of a product ("linear", "gated", "dx" or
    "dw") of torch types; out_dtype is dtype (bfloat16 for e4m3) unless given."""
    products, codes = ("linear", "gated", "dx", "dw"), _dtype_codes()
    if product not in products:
        _invalid(f"unknown product {product!r}")
    for d in (dtype, out_dtype):
        if d is not None and d not in codes:
            _invalid(f"no such element type: {d}")
    t = codes[dtype]
    out = codes[out_dtype] if out_dtype is not None else abi.BF16 if t == abi.E4M3 else t
    launches = (LinearLaunch * 2)()
    check(lib().jh_op_linear_plan(products.index(product), t, out, rows, n, k, launches))
    names = ("small", "deep", "pair", "tall", "wide", "stream")
    return [(names[v.kernel], v.parts, v.rows) for v in launches if v.parts]


def op_gated_ffn(x, wi, out, act="gelu", x_scale=None, w_scale=None, gu=None, stream=None):
    """jh_op_gated_ffn: out = act(x Wg^T) * (x Wu^T), wi = [Wg; Wu]; types as op_linear (out of x's type, bf16 for
    e4m3); gu [rows, 2 inter] keeps both projections for the backward."""
    xp, ldx, (rows, k), dev = _first("x", x)
    n, dt, code = wi.shape[0], x.dtype, _type(x)
    if n % 2:
        _invalid("wi: needs an even number of rows")
    if _type(out) != (abi.BF16 if code == abi.E4M3 else code):
        _invalid("out: has x's type (bfloat16 for e4m3)")
    op, ldo = _mat("out", out, (rows, n // 2), dev, out.dtype)
    gp = xs = ws = None
    ldg = 0
    if gu is not None:
        gp, ldg = _mat("gu", gu, (rows, n), dev, dt)
    if x_scale is not None:
        xs = _vec("x_scale", x_scale, rows, dev)
    if w_scale is not None:
        ws = _vec("w_scale", w_scale, n, dev)
    check(lib().jh_op_gated_ffn(code, xp, ldx, xs, rows, _weight("wi", wi, (n, k), dev, dt), ws, n // 2, k, _act(act), op,
                                ldo, gp, ldg, stream))


def op_gated_ffn_backward(dh, gu, x, wi, workspace, act="gelu", dx=None, dw=None, stream=None):
    """jh_op_gated_ffn_backward: dx and / or dw (of wi; f32 or x's type) from dh and gu; workspace of
    gated_ffn_backward_workspace(rows, inter, k) bytes."""
    hp, ldh, (rows, inter), dev = _first("dh", dh)
    k, n, dt = wi.shape[1], 2 * inter, dh.dtype
    gp, ldg = _mat("gu", gu, (rows, n), dev, dt)
    (xp, ldx), (dp, ldd) = _mat("x", x, (rows, k), dev, dt), _mat("dx", dx, (rows, k), dev, dt)
    wp, wb = _space(workspace, dev)
    check(lib().jh_op_gated_ffn_backward(_type(dh), hp, ldh, gp, ldg, xp, ldx, rows, _weight("wi", wi, (n, k), dev, dt),
                                         inter, k, _act(act), dp, ldd, _type(dh if dw is None else dw),
                                         _weight("dw", dw, (n, k), dev, dt if dw is None else dw.dtype), wp, wb, stream))


def gated_ffn_backward_workspace(rows, inter, k) -> int:
    return _bytes(lib().jh_op_gated_ffn_backward_workspace(rows, inter, k))
