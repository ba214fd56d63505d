"""ctypes binding of the B200 C-ABI library (``libr4c_conv3d.so``).

This module is the only place Python touches the native kernels. It is the
reference-side binding of ``include/r4c_conv3d.h``: it turns torch tensors into
plain pointers and sizes, passes torch's current CUDA stream, and turns status
codes into exceptions. There is deliberately no host fallback: if the library
is missing or the call fails, the caller gets an exception.

Reference counterpart: the JIT loader of the HIP extension
(src/rdna4_conv3d/hip_backend.py:1-37) and the Triton launchers it sat next to
(src/rdna4_conv3d/conv3d_wmma.py:1015-1227, 1453-1542).
"""
from __future__ import annotations

import ctypes
import functools
import os
import threading
from typing import Optional, Tuple

import torch

_LIB_NAME = "libr4c_conv3d.so"
_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), _LIB_NAME)
_lib = None
_lock = threading.Lock()

# Must match include/r4c_conv3d.h.
R4C_OK = 0
R4C_BF16, R4C_F16, R4C_F32 = 0, 1, 2
LEG_FWD, LEG_DX, LEG_DW, LEG_TFWD, LEG_TDX, LEG_TDW = range(6)
KERNEL_NONE, KERNEL_GENERIC, KERNEL_TC = 0, 1, 2


class ConvDesc(ctypes.Structure):
    _fields_ = [
        ("n", ctypes.c_int32), ("d", ctypes.c_int32), ("h", ctypes.c_int32), ("w", ctypes.c_int32),
        ("cin", ctypes.c_int32), ("cout", ctypes.c_int32), ("k", ctypes.c_int32),
        ("pad_d", ctypes.c_int32), ("pad_h", ctypes.c_int32), ("pad_w", ctypes.c_int32),
        ("dtype", ctypes.c_int32), ("force_kernel", ctypes.c_int32),
    ]


class ConvexDesc(ctypes.Structure):
    """r4c_convex_desc: Conv3d of any geometry (include/r4c_conv3d.h)."""
    _fields_ = [(name, ctypes.c_int32) for name in (
        "n", "d", "h", "w", "cin", "cout", "groups", "kd", "kh", "kw", "sd", "sh", "sw",
        "pd", "ph", "pw", "dd", "dh", "dw", "dtype")]


class RowsDesc(ctypes.Structure):
    """r4c_rows_desc: rows of logits (include/r4c_conv3d.h)."""
    _fields_ = [("rows", ctypes.c_int64), ("inner", ctypes.c_int64),
                ("outer_stride", ctypes.c_int64), ("inner_stride", ctypes.c_int64), ("class_stride", ctypes.c_int64),
                ("grad_outer_stride", ctypes.c_int64), ("grad_inner_stride", ctypes.c_int64),
                ("grad_class_stride", ctypes.c_int64),
                ("classes", ctypes.c_int32), ("dtype", ctypes.c_int32), ("temperature", ctypes.c_float)]


class GnDesc(ctypes.Structure):
    """r4c_gn_desc: channels-last activations in groups (include/r4c_conv3d.h)."""
    _fields_ = [("samples", ctypes.c_int64), ("inner", ctypes.c_int64),
                ("channels", ctypes.c_int32), ("groups", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("param_dtype", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("eps", ctypes.c_float), ("slope", ctypes.c_float)]


class NativeError(RuntimeError):
    """A C-ABI entry point returned a non-zero status."""


def library_path() -> str:
    return _LIB_PATH


def _bind(lib) -> None:
    P = ctypes.c_void_p
    D = ctypes.POINTER(ConvDesc)
    X = ctypes.POINTER(ConvexDesc)
    R = ctypes.POINTER(RowsDesc)
    N = ctypes.POINTER(GnDesc)
    sz = ctypes.c_size_t
    i = ctypes.c_int
    i64 = ctypes.c_int64
    dbl = ctypes.c_double
    flt = ctypes.c_float
    sig = {
        "r4c_strerror": ([i], ctypes.c_char_p),
        "r4c_version": ([], i),
        "r4c_device_error": ([P, i], i),
        "r4c_watchdog_selftest": ([ctypes.c_uint64, P], i),
        "r4c_launch_count": ([], ctypes.c_uint64),
        "r4c_plan_kernel": ([D, i], i),
        "r4c_describe_plan": ([D, i, ctypes.c_char_p, sz], i),
        "r4c_packed_weight_bytes": ([D, i], sz),
        "r4c_workspace_size": ([D, i], sz),
        "r4c_pack_weight": ([D, i, P, i, P, P], i),
        "r4c_conv3d_fwd": ([D, P, P, P, P, P, sz, P], i),
        "r4c_conv3d_dx": ([D, P, P, P, P, sz, P], i),
        "r4c_conv3d_dw": ([D, P, P, P, P, P, sz, P], i),
        "r4c_tconv_fwd": ([D, P, P, P, P, P, sz, P], i),
        "r4c_tconv_fwd_pitched": ([D, P, P, P, P, i, P, sz, P], i),
        "r4c_tconv_dx": ([D, P, P, P, P, sz, P], i),
        "r4c_tconv_dw": ([D, P, P, P, P, P, sz, P], i),
        "r4c_bn_workspace_size": ([i64, i], sz),
        "r4c_bn_stats": ([P, i64, i, i, P, P, P, sz, P], i),
        "r4c_bn_finalize": ([P, dbl, i, P, P, flt, flt, P, P, P, P, P], i),
        "r4c_bn_relu_fwd": ([P, P, P, P, i64, i, i, i, P], i),
        "r4c_bn_relu_bwd_sums": ([P, P, P, P, i64, i, i, i, P, P, sz, P], i),
        "r4c_bn_relu_bwd_dx": ([P, P, P, P, P, P, dbl, i64, i, i, i, P, P, P, P], i),
        "r4c_channel_slice_copy": ([P, i, P, i64, i, i, P], i),
        "r4c_bn_relu_pool_fwd": ([P, P, i, P, P, P, i, i, i, i, i, i, P], i),
        "r4c_bn_relu_pool_fwd_cat": ([P, P, i, P, P, P, P, i, i, i, i, i, i, P], i),
        "r4c_bn_pool_workspace_size": ([i, i, i, i, i], sz),
        "r4c_bn_relu_pool_bwd_sums": ([P, i, P, P, P, P, P, i, i, i, i, i, i, P, P, sz, P], i),
        "r4c_bn_relu_pool_bwd_dx": ([P, i, P, P, P, P, P, P, P, dbl, i, i, i, i, i, i, P, P, P, P], i),
        "r4c_ce_workspace_size": ([i64], sz),
        "r4c_ce_fwd": ([P, P, i64, i, i, i64, P, P, sz, P], i),
        "r4c_ce_bwd": ([P, P, i64, i, i, i64, P, P, P, P], i),
        "r4c_logp_stats_size": ([R], sz),
        "r4c_logp_fwd": ([R, P, P, i64, i, P, P, P, P, P, P, P], i),
        "r4c_logp_bwd": ([R, P, P, i64, P, P, P, i, P, i, P, i, P, P], i),
        "r4c_distill_state_size": ([R], sz),
        "r4c_distill_fwd": ([R, P, i, P, i, P, i, i, P, P, P, P, sz, P], i),
        "r4c_distill_bwd": ([R, P, i, P, i, P, i, i, P, i, P, i, P, P, P], i),
        "r4c_pack8": ([P, i64, i, i, P, P, P], i),
        "r4c_unpack8": ([P, P, i64, i, i, P, P], i),
        "r4c_gn_workspace_size": ([N, i], sz),
        "r4c_gn_fwd": ([N, P, P, P, P, P, i, P, P, P, sz, P], i),
        "r4c_gn_bwd": ([N, P, P, i, P, P, P, P, P, P, P, P, sz, P], i),
        "r4c_convex_plan": ([X], i),
        "r4c_convex_workspace_size": ([X, i], sz),
        "r4c_convex_fwd": ([X, P, P, P, P, P, sz, P], i),
        "r4c_convex_dx": ([X, P, P, P, P, sz, P], i),
        "r4c_convex_dw": ([X, P, P, P, P, P, sz, P], i),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res


def lib():
    """Load (once) and return the native library; raise if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(_LIB_PATH):
                raise NativeError(
                    f"rdna4_conv3d native library not built: {_LIB_PATH} is missing "
                    "(run `python -m rdna4_conv3d.build` or __graft_entry__.build())")
            handle = ctypes.CDLL(_LIB_PATH)
            _bind(handle)
            _lib = handle
    return _lib


def available() -> bool:
    try:
        lib()
        return True
    except (NativeError, OSError):
        return False


def strerror(status: int) -> str:
    return lib().r4c_strerror(int(status)).decode()


def _check(status: int, what: str) -> None:
    if status != R4C_OK:
        raise NativeError(f"{what} failed: {strerror(status)} (status {status})")


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return R4C_BF16
    if dt == torch.float16:
        return R4C_F16
    if dt == torch.float32:
        return R4C_F32
    raise NativeError(f"unsupported dtype {dt}")


def make_desc(n, d, h, w, cin, cout, k, pad, dtype: torch.dtype, force_kernel: int = 0) -> ConvDesc:
    pd, ph, pw = pad
    return ConvDesc(int(n), int(d), int(h), int(w), int(cin), int(cout), int(k),
                    int(pd), int(ph), int(pw), dtype_code(dtype), int(force_kernel))


def _stream(device: torch.device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _require_cuda(*ts: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise NativeError("rdna4_conv3d native kernels need CUDA tensors")
        dev = t.device if dev is None else dev
    return dev


def plan_kernel(desc: ConvDesc, leg: int) -> int:
    return int(lib().r4c_plan_kernel(ctypes.byref(desc), leg))


def describe_plan(desc: ConvDesc, leg: int) -> str:
    buf = ctypes.create_string_buffer(512)
    lib().r4c_describe_plan(ctypes.byref(desc), leg, buf, 512)
    return buf.value.decode()


def workspace_bytes(desc: ConvDesc, leg: int) -> int:
    return int(lib().r4c_workspace_size(ctypes.byref(desc), leg))


def packed_weight_bytes(desc: ConvDesc, leg: int) -> int:
    return int(lib().r4c_packed_weight_bytes(ctypes.byref(desc), leg))


def _workspace(desc: ConvDesc, leg: int, device) -> Tuple[Optional[torch.Tensor], int]:
    nb = workspace_bytes(desc, leg)
    if nb == 0:
        return None, 0
    return torch.empty(nb, dtype=torch.uint8, device=device), nb


def pack_weight(desc: ConvDesc, leg: int, weight: torch.Tensor) -> torch.Tensor:
    """Pack a PyTorch-layout weight for one leg (r4c_pack_weight)."""
    dev = _require_cuda(weight)
    w = weight.contiguous()
    nbytes = packed_weight_bytes(desc, leg)
    if nbytes == 0:
        raise NativeError("descriptor rejected by r4c_packed_weight_bytes")
    out = torch.empty(nbytes // 2, dtype=torch.bfloat16 if desc.dtype == R4C_BF16 else torch.float16,
                      device=dev)
    with torch.cuda.device(dev):
        st = lib().r4c_pack_weight(ctypes.byref(desc), leg, _ptr(w), dtype_code(w.dtype), _ptr(out),
                                   _stream(dev))
    _check(st, "r4c_pack_weight")
    return out


def _ndhwc_empty(n, c, d, h, w, device, dtype) -> torch.Tensor:
    return torch.empty((n, c, d, h, w), device=device, dtype=dtype, memory_format=torch.channels_last_3d)


def _check_out(out: torch.Tensor, shape, dtype) -> torch.Tensor:
    """A caller-given output must be a dense NDHWC buffer of the right size."""
    if (tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_cuda
            or not out.is_contiguous(memory_format=torch.channels_last_3d) or out.data_ptr() % 16):
        raise NativeError(f"out must be a 16-byte aligned channels_last_3d {dtype} tensor of shape {tuple(shape)}")
    return out


def conv_fwd(desc: ConvDesc, x_cl: torch.Tensor, w_packed: torch.Tensor, bias: Optional[torch.Tensor],
             out_shape, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    dev = _require_cuda(x_cl, w_packed, bias)
    od, oh, ow = out_shape
    if out is None:
        y = _ndhwc_empty(desc.n, desc.cout, od, oh, ow, dev, x_cl.dtype)
    else:
        y = _check_out(out, (desc.n, desc.cout, od, oh, ow), x_cl.dtype)
    ws, nb = _workspace(desc, LEG_FWD, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_conv3d_fwd(ctypes.byref(desc), _ptr(x_cl), _ptr(w_packed), _ptr(bias), _ptr(y),
                                  _ptr(ws), nb, _stream(dev))
    _check(st, "r4c_conv3d_fwd")
    return y


def conv_dx(desc: ConvDesc, go_cl: torch.Tensor, w_packed: torch.Tensor,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    dev = _require_cuda(go_cl, w_packed)
    if out is None:
        dx = _ndhwc_empty(desc.n, desc.cin, desc.d, desc.h, desc.w, dev, go_cl.dtype)
    else:
        dx = _check_out(out, (desc.n, desc.cin, desc.d, desc.h, desc.w), go_cl.dtype)
    ws, nb = _workspace(desc, LEG_DX, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_conv3d_dx(ctypes.byref(desc), _ptr(go_cl), _ptr(w_packed), _ptr(dx), _ptr(ws), nb,
                                 _stream(dev))
    _check(st, "r4c_conv3d_dx")
    return dx


def conv_dw(desc: ConvDesc, x_cl: torch.Tensor, go_cl: torch.Tensor, want_db: bool):
    """fp32 OIDHW weight gradient and (optionally) fp32 bias gradient."""
    dev = _require_cuda(x_cl, go_cl)
    k = desc.k
    dw = torch.empty((desc.cout, desc.cin, k, k, k), dtype=torch.float32, device=dev)
    db = torch.empty((desc.cout,), dtype=torch.float32, device=dev) if want_db else None
    ws, nb = _workspace(desc, LEG_DW, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_conv3d_dw(ctypes.byref(desc), _ptr(x_cl), _ptr(go_cl), _ptr(dw), _ptr(db), _ptr(ws), nb,
                                 _stream(dev))
    _check(st, "r4c_conv3d_dw")
    return dw, db


def tconv_fwd(desc: ConvDesc, x_cl: torch.Tensor, w_packed: torch.Tensor,
              bias: Optional[torch.Tensor]) -> torch.Tensor:
    dev = _require_cuda(x_cl, w_packed, bias)
    y = _ndhwc_empty(desc.n, desc.cout, 2 * desc.d, 2 * desc.h, 2 * desc.w, dev, x_cl.dtype)
    ws, nb = _workspace(desc, LEG_TFWD, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_tconv_fwd(ctypes.byref(desc), _ptr(x_cl), _ptr(w_packed), _ptr(bias), _ptr(y),
                                 _ptr(ws), nb, _stream(dev))
    _check(st, "r4c_tconv_fwd")
    return y


def tconv_fwd_into(desc: ConvDesc, x_cl: torch.Tensor, w_packed: torch.Tensor, bias: Optional[torch.Tensor],
                   buf: torch.Tensor) -> None:
    """The transpose conv's output written into channels [0, Cout) of ``buf``,
    a dense NDHWC buffer with more channels (r4c_tconv_fwd_pitched)."""
    dev = _require_cuda(x_cl, w_packed, bias, buf)
    pitch = int(buf.shape[1])
    if (tuple(buf.shape) != (desc.n, pitch, 2 * desc.d, 2 * desc.h, 2 * desc.w) or buf.dtype != x_cl.dtype
            or not buf.is_contiguous(memory_format=torch.channels_last_3d) or buf.data_ptr() % 16 or pitch < desc.cout):
        raise NativeError("buf must be a 16-byte aligned channels_last_3d tensor (N, >= Cout, 2D, 2H, 2W) of x's dtype")
    ws, nb = _workspace(desc, LEG_TFWD, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_tconv_fwd_pitched(ctypes.byref(desc), _ptr(x_cl), _ptr(w_packed), _ptr(bias), _ptr(buf),
                                         pitch, _ptr(ws), nb, _stream(dev))
    _check(st, "r4c_tconv_fwd_pitched")


def tconv_dx(desc: ConvDesc, go_cl: torch.Tensor, w_packed: torch.Tensor) -> torch.Tensor:
    dev = _require_cuda(go_cl, w_packed)
    dx = _ndhwc_empty(desc.n, desc.cin, desc.d, desc.h, desc.w, dev, go_cl.dtype)
    ws, nb = _workspace(desc, LEG_TDX, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_tconv_dx(ctypes.byref(desc), _ptr(go_cl), _ptr(w_packed), _ptr(dx), _ptr(ws), nb,
                                _stream(dev))
    _check(st, "r4c_tconv_dx")
    return dx


def tconv_dw(desc: ConvDesc, x_cl: torch.Tensor, go_cl: torch.Tensor, want_db: bool):
    dev = _require_cuda(x_cl, go_cl)
    dw = torch.empty((desc.cin, desc.cout, 2, 2, 2), dtype=torch.float32, device=dev)
    db = torch.empty((desc.cout,), dtype=torch.float32, device=dev) if want_db else None
    ws, nb = _workspace(desc, LEG_TDW, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_tconv_dw(ctypes.byref(desc), _ptr(x_cl), _ptr(go_cl), _ptr(dw), _ptr(db), _ptr(ws), nb,
                                _stream(dev))
    _check(st, "r4c_tconv_dw")
    return dw, db


# ---------------------------------------------------------------------------
# Conv3d of any geometry (r4c_convex_*)
# ---------------------------------------------------------------------------
def make_convex_desc(x_shape, w_shape, stride, padding, dilation, groups, dtype: torch.dtype) -> ConvexDesc:
    n, cin, d, h, w = (int(v) for v in x_shape)
    cout, _, kd, kh, kw = (int(v) for v in w_shape)
    return ConvexDesc(n, d, h, w, cin, cout, int(groups), kd, kh, kw, *(int(v) for v in stride),
                      *(int(v) for v in padding), *(int(v) for v in dilation), dtype_code(dtype))


def convex_out_shape(desc: ConvexDesc):
    o = lambda i, k, s, p, dl: (i + 2 * p - dl * (k - 1) - 1) // s + 1  # noqa: E731
    return (desc.n, desc.cout, o(desc.d, desc.kd, desc.sd, desc.pd, desc.dd), o(desc.h, desc.kh, desc.sh, desc.ph, desc.dh),
            o(desc.w, desc.kw, desc.sw, desc.pw, desc.dw))


def convex_plan(desc: ConvexDesc) -> int:
    return int(lib().r4c_convex_plan(ctypes.byref(desc)))


def _convex_ws(desc: ConvexDesc, leg: int, device):
    nb = int(lib().r4c_convex_workspace_size(ctypes.byref(desc), leg))
    if nb == 0:
        return None, 0
    return torch.empty(nb, dtype=torch.uint8, device=device), nb


def convex_fwd(desc: ConvexDesc, x_cl: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    dev = _require_cuda(x_cl, w, bias)
    shp = convex_out_shape(desc)
    y = _ndhwc_empty(*shp, dev, x_cl.dtype)
    ws, nb = _convex_ws(desc, LEG_FWD, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_convex_fwd(ctypes.byref(desc), _ptr(x_cl), _ptr(w), _ptr(bias), _ptr(y), _ptr(ws), nb,
                                  _stream(dev))
    _check(st, "r4c_convex_fwd")
    return y


def convex_dx(desc: ConvexDesc, go_cl: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    dev = _require_cuda(go_cl, w)
    dx = _ndhwc_empty(desc.n, desc.cin, desc.d, desc.h, desc.w, dev, go_cl.dtype)
    ws, nb = _convex_ws(desc, LEG_DX, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_convex_dx(ctypes.byref(desc), _ptr(go_cl), _ptr(w), _ptr(dx), _ptr(ws), nb, _stream(dev))
    _check(st, "r4c_convex_dx")
    return dx


def convex_dw(desc: ConvexDesc, x_cl: torch.Tensor, go_cl: torch.Tensor, want_db: bool):
    dev = _require_cuda(x_cl, go_cl)
    dw = torch.empty((desc.cout, desc.cin // desc.groups, desc.kd, desc.kh, desc.kw), dtype=torch.float32, device=dev)
    db = torch.empty((desc.cout,), dtype=torch.float32, device=dev) if want_db else None
    ws, nb = _convex_ws(desc, LEG_DW, dev)
    with torch.cuda.device(dev):
        st = lib().r4c_convex_dw(ctypes.byref(desc), _ptr(x_cl), _ptr(go_cl), _ptr(dw), _ptr(db), _ptr(ws), nb,
                                 _stream(dev))
    _check(st, "r4c_convex_dw")
    return dw, db


# ---------------------------------------------------------------------------
# BatchNorm3d + ReLU (r4c_bn_*)
# ---------------------------------------------------------------------------
def bn_relu_forward(x_cl: torch.Tensor, gamma, beta, running_mean, running_var, momentum: float, eps: float,
                    relu: bool, sums_hook=None, pivot=None, apply: bool = True):
    """Training forward. Returns (y, mean_invstd, affine, count).
    ``sums_hook(sums, count)``, when given, may all-reduce the per-channel
    sums in place before they are finalised and returns the total count (a
    volume sharded over ranks: every rank then passes the same ``pivot``)."""
    dev = _require_cuda(x_cl)
    C = int(x_cl.shape[1])
    vox = x_cl.numel() // C
    L = lib()
    f32 = dict(dtype=torch.float32, device=dev)
    ws = torch.empty(int(L.r4c_bn_workspace_size(vox, C)), dtype=torch.uint8, device=dev)
    sums = torch.empty(3 * C, **f32)
    mi = torch.empty(2 * C, **f32)
    ss = torch.empty(2 * C, **f32)
    y = torch.empty_like(x_cl, memory_format=torch.channels_last_3d) if apply else None
    dt = dtype_code(x_cl.dtype)
    with torch.cuda.device(dev):
        st = L.r4c_bn_stats(_ptr(x_cl), vox, C, dt, _ptr(pivot), _ptr(sums), _ptr(ws), ws.numel(), _stream(dev))
        _check(st, "r4c_bn_stats")
        count = float(vox)
        if sums_hook is not None:
            count = float(sums_hook(sums, count))
        st = L.r4c_bn_finalize(_ptr(sums), count, C, _ptr(gamma), _ptr(beta), float(eps), float(momentum),
                               _ptr(running_mean), _ptr(running_var), _ptr(mi), _ptr(ss), _stream(dev))
        _check(st, "r4c_bn_finalize")
        if apply:
            st = L.r4c_bn_relu_fwd(_ptr(x_cl), _ptr(y), _ptr(mi), _ptr(ss), vox, C, dt, 1 if relu else 0,
                                   _stream(dev))
            _check(st, "r4c_bn_relu_fwd")
    return (y if apply else None), mi, ss, count


def bn_relu_backward(dy_cl: torch.Tensor, x_cl: torch.Tensor, mean_invstd, affine, count: float, relu: bool,
                     need_dx: bool = True, sums_hook=None):
    """(dx or None, dgamma, dbeta), fp32 parameter gradients."""
    dev = _require_cuda(dy_cl, x_cl)
    C = int(x_cl.shape[1])
    vox = x_cl.numel() // C
    L = lib()
    f32 = dict(dtype=torch.float32, device=dev)
    ws = torch.empty(int(L.r4c_bn_workspace_size(vox, C)), dtype=torch.uint8, device=dev)
    sums = torch.empty(2 * C, **f32)
    dg = torch.empty(C, **f32)
    db = torch.empty(C, **f32)
    coef = torch.empty(3 * C, **f32)
    dx = torch.empty_like(x_cl, memory_format=torch.channels_last_3d) if need_dx else None
    dt = dtype_code(x_cl.dtype)
    with torch.cuda.device(dev):
        st = L.r4c_bn_relu_bwd_sums(_ptr(dy_cl), _ptr(x_cl), _ptr(mean_invstd), _ptr(affine), vox, C, dt,
                                    1 if relu else 0, _ptr(sums), _ptr(ws), ws.numel(), _stream(dev))
        _check(st, "r4c_bn_relu_bwd_sums")
        if sums_hook is not None:
            sums_hook(sums, None)
        st = L.r4c_bn_relu_bwd_dx(_ptr(dy_cl), _ptr(x_cl), _ptr(dx), _ptr(mean_invstd), _ptr(affine),
                                  _ptr(sums), float(count), vox, C, dt, 1 if relu else 0, _ptr(dg), _ptr(db),
                                  _ptr(coef), _stream(dev))
        _check(st, "r4c_bn_relu_bwd_dx")
    return dx, dg, db


def channel_slice_dense(t: torch.Tensor) -> Optional[torch.Tensor]:
    """A dense channels_last_3d copy of ``t`` when ``t`` is a channel slice of
    a wider NDHWC tensor (voxel stride = pitch >= C, channel stride 1), made
    by the library's slice copy; None when ``t`` is not such a slice or the
    copy's alignment rules do not hold."""
    if t.dim() != 5 or not t.is_cuda or t.dtype not in (torch.bfloat16, torch.float16):
        return None
    n, C, d, h, w = (int(v) for v in t.shape)
    sn, sc, sd, sh, sw = t.stride()
    pitch = sw
    if (sc != 1 or C % 8 or pitch % 8 or pitch < C or sh != pitch * w or sd != pitch * w * h
            or (n > 1 and sn != pitch * w * h * d) or t.data_ptr() % 16):
        return None
    dev = t.device
    out = _ndhwc_empty(n, C, d, h, w, dev, t.dtype)
    with torch.cuda.device(dev):
        st = lib().r4c_channel_slice_copy(_ptr(t), pitch, _ptr(out), n * d * h * w, C, dtype_code(t.dtype),
                                          _stream(dev))
    _check(st, "r4c_channel_slice_copy")
    return out


def bn_relu_pool_forward(x_cl: torch.Tensor, mean_invstd, affine, lead: int):
    """(buf, p, argmax): buf is a new NDHWC tensor of lead + C channels whose
    channels [lead, lead + C) hold relu(bn(x)) (the first lead channels zero
    when lead is a multiple of 8, else unwritten: the caller's), p the 2x2x2
    max-pool of those channels, argmax the windows' argmax for the backward
    (int16 storage of the uint16 fields; None when lead is not a multiple of 8)."""
    dev = _require_cuda(x_cl)
    n, C, d, h, w = (int(v) for v in x_cl.shape)
    buf = _ndhwc_empty(n, lead + C, d, h, w, dev, x_cl.dtype)
    p = _ndhwc_empty(n, C, d // 2, h // 2, w // 2, dev, x_cl.dtype)
    am = None
    with torch.cuda.device(dev):
        if lead % 8 == 0:
            # whole voxels in one pass (channels [0, lead) zero until the up-conv writes them)
            am = torch.empty(n * (d // 2) * (h // 2) * (w // 2) * (C // 4), dtype=torch.int16, device=dev)
            st = lib().r4c_bn_relu_pool_fwd_cat(_ptr(x_cl), _ptr(buf), lead, _ptr(p), _ptr(am), _ptr(mean_invstd),
                                                _ptr(affine), n, d, h, w, C, dtype_code(x_cl.dtype), _stream(dev))
        else:
            yptr = ctypes.c_void_p(buf.data_ptr() + lead * buf.element_size())
            st = lib().r4c_bn_relu_pool_fwd(_ptr(x_cl), yptr, lead + C, _ptr(p), _ptr(mean_invstd), _ptr(affine),
                                            n, d, h, w, C, dtype_code(x_cl.dtype), _stream(dev))
    _check(st, "r4c_bn_relu_pool_fwd")
    return buf, p, am


def bn_relu_pool_backward(gbuf_cl: torch.Tensor, lead: int, gp_cl: torch.Tensor, x_cl: torch.Tensor, mean_invstd,
                          affine, count: float, need_dx: bool = True, sums_hook=None, argmax=None):
    """(dx or None, dgamma, dbeta) from dY = channels [lead, lead + C) of gbuf
    and dP = gp; argmax: the forward's (None: recomputed from x)."""
    dev = _require_cuda(gbuf_cl, gp_cl, x_cl)
    n, C, d, h, w = (int(v) for v in x_cl.shape)
    L = lib()
    f32 = dict(dtype=torch.float32, device=dev)
    ws = torch.empty(int(L.r4c_bn_pool_workspace_size(n, d, h, w, C)), dtype=torch.uint8, device=dev)
    sums = torch.empty(2 * C, **f32)
    dg = torch.empty(C, **f32)
    db = torch.empty(C, **f32)
    coef = torch.empty(3 * C, **f32)
    dx = _ndhwc_empty(n, C, d, h, w, dev, x_cl.dtype) if need_dx else None
    dt = dtype_code(x_cl.dtype)
    pitch = int(gbuf_cl.shape[1])
    gyptr = ctypes.c_void_p(gbuf_cl.data_ptr() + lead * gbuf_cl.element_size())
    with torch.cuda.device(dev):
        st = L.r4c_bn_relu_pool_bwd_sums(gyptr, pitch, _ptr(gp_cl), _ptr(argmax), _ptr(x_cl), _ptr(mean_invstd),
                                         _ptr(affine),
                                         n, d, h, w, C, dt, _ptr(sums), _ptr(ws), ws.numel(), _stream(dev))
        _check(st, "r4c_bn_relu_pool_bwd_sums")
        if sums_hook is not None:
            sums_hook(sums, None)
        st = L.r4c_bn_relu_pool_bwd_dx(gyptr, pitch, _ptr(gp_cl), _ptr(argmax), _ptr(x_cl), _ptr(dx),
                                       _ptr(mean_invstd),
                                       _ptr(affine), _ptr(sums), float(count), n, d, h, w, C, dt, _ptr(dg), _ptr(db),
                                       _ptr(coef), _stream(dev))
        _check(st, "r4c_bn_relu_pool_bwd_dx")
    return dx, dg, db


def launch_count() -> int:
    """Kernels launched by the native library so far in this process."""
    return int(lib().r4c_launch_count())


def watchdog_selftest(limit_ns: int, device=None) -> None:
    """Launch the bounded-wait self-test (a wait that runs out after limit_ns)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        _check(lib().r4c_watchdog_selftest(int(limit_ns), _stream(dev)), "r4c_watchdog_selftest")


def device_error(device=None, clear: bool = True) -> int:
    """Read (and clear) the kernels' device-side timeout flag."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        return int(lib().r4c_device_error(_stream(dev), 1 if clear else 0))


# ---------------------------------------------------------------------------
# Cross-entropy over NDHWC logits (r4c_ce_*)
# ---------------------------------------------------------------------------
def ce_forward(logits_cl: torch.Tensor, target: torch.Tensor, ignore_index: int) -> torch.Tensor:
    """(mean loss, counted voxels) as a 2-float device tensor."""
    dev = _require_cuda(logits_cl, target)
    C = int(logits_cl.shape[1])
    vox = logits_cl.numel() // C
    L = lib()
    ws = torch.empty(int(L.r4c_ce_workspace_size(vox)), dtype=torch.uint8, device=dev)
    out = torch.empty(2, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        st = L.r4c_ce_fwd(_ptr(logits_cl), _ptr(target), vox, C, dtype_code(logits_cl.dtype), int(ignore_index),
                          _ptr(out), _ptr(ws), ws.numel(), _stream(dev))
    _check(st, "r4c_ce_fwd")
    return out


def ce_backward(logits_cl: torch.Tensor, target: torch.Tensor, ignore_index: int, loss_count: torch.Tensor,
                grad: torch.Tensor) -> torch.Tensor:
    """d(loss)/d(logits), NDHWC in the logits' dtype; ``grad`` a device scalar."""
    dev = _require_cuda(logits_cl, target)
    C = int(logits_cl.shape[1])
    vox = logits_cl.numel() // C
    g = grad.detach().to(torch.float32).reshape(1).contiguous()
    dz = torch.empty_like(logits_cl, memory_format=torch.channels_last_3d)
    with torch.cuda.device(dev):
        st = lib().r4c_ce_bwd(_ptr(logits_cl), _ptr(target), vox, C, dtype_code(logits_cl.dtype), int(ignore_index),
                              _ptr(loss_count), _ptr(g), _ptr(dz), _stream(dev))
    _check(st, "r4c_ce_bwd")
    return dz


# ---------------------------------------------------------------------------
# Rows of logits: log-probabilities (r4c_logp_*), distillation (r4c_distill_*)
# ---------------------------------------------------------------------------
TOPK_MAX = 128
# Rows up to this many classes are read with any class stride; wider ones are
# copied class-last first (105 bf16 classes laid out class first: 193 + 62 us
# forward + backward with the copy, 102 + 187 us gathered; 300 classes: 647 +
# 206 against 858 + 1650 us).
_TILE_CLASSES = 32


def _row_strides(t: torch.Tensor):
    """(inner, outer stride, inner stride, class stride) of (N, C, ...) logits
    whose dims after the class walk one stride; None when they do not."""
    n, c = int(t.shape[0]), int(t.shape[1])
    if t.numel() == 0:                   # no rows: nothing to walk
        return 1, 0, c, 1
    st = t.stride()
    inner, si = 1, 0
    for size, stride in zip(reversed(t.shape[2:]), reversed(st[2:])):
        if size == 1:
            continue
        if inner == 1:
            si = stride
        elif stride != si * inner:
            return None
        inner *= int(size)
    sc = st[1] if c > 1 else 1
    if inner == 1:                       # rows are the outer dim
        return max(n, 1), 0, st[0] if n > 1 else c, sc
    if n == 1 or st[0] == si * inner:    # one stride over everything
        return n * inner, 0, si, sc
    return inner, st[0], si, sc


def class_last_empty(t: torch.Tensor) -> torch.Tensor:
    """A new tensor of t's shape whose memory order puts the classes (dim 1) last."""
    shape = t.shape
    return torch.empty((shape[0], *shape[2:], shape[1]), dtype=t.dtype, device=t.device).movedim(-1, 1)


class Rows:
    """Logits as the row kernels read them: ``z`` (the logits themselves, or a
    class-last copy where the kernels cannot walk their strides), their
    descriptor, and the per-row shape (N, ...)."""
    __slots__ = ("z", "desc", "shape")

    def __init__(self, logits: torch.Tensor, temperature: float):
        z = logits
        shape = z.shape
        c = shape[1]
        if len(shape) == 2 and z.is_contiguous():
            n = shape[0]
            inner, so, si, sc = n or 1, 0, c, 1
            self.shape = shape[:1]
        else:
            st = _row_strides(z)
            if st is None or (st[3] != 1 and c > _TILE_CLASSES):
                z = class_last_empty(logits).copy_(logits)
                st = _row_strides(z)
            inner, so, si, sc = st
            self.shape = shape[:1] + shape[2:]
            n = self.shape.numel()
        self.z = z
        self.desc = RowsDesc(n, inner or 1, so, si, sc, so, si, sc, c, dtype_code(z.dtype), temperature)


class SavedRows:
    """What a backward knows of its forward's rows beside the tensors it saved.
    A saved tensor may come back as another one with the same values (hooks
    that offload or pack what autograd keeps): other strides get a descriptor
    of their own, another shape, type or device never reaches a kernel."""
    __slots__ = ("desc", "shape", "stride", "dtype", "device")

    def __init__(self, rows: Rows):
        z = rows.z
        self.desc, self.shape, self.stride, self.dtype, self.device = rows.desc, z.shape, z.stride(), z.dtype, z.device

    def logits(self, z: torch.Tensor):
        """(logits as the kernels read them, their descriptor)."""
        if z.shape != self.shape or z.dtype is not self.dtype or z.device != self.device:
            _not_as_saved(z, self.shape, self.dtype, self.device)
        if z.stride() == self.stride:
            return z, self.desc
        rows = Rows(z, self.desc.temperature)
        return rows.z, rows.desc

    def dense(self, t: torch.Tensor, shape, dtype: torch.dtype) -> torch.Tensor:
        """A per-row tensor of this shape as the kernels read it."""
        if t.shape != shape or t.dtype is not dtype or t.device != self.device:
            _not_as_saved(t, shape, dtype, self.device)
        return t if t.is_contiguous() else t.contiguous()

    def buffer(self, t: torch.Tensor, nbytes: int) -> torch.Tensor:
        """A forward's own bytes for its backward, 16-byte aligned."""
        if t.numel() != nbytes or t.dtype is not torch.uint8 or t.device != self.device:
            _not_as_saved(t, (nbytes,), torch.uint8, self.device)
        if not t.is_contiguous() or t.data_ptr() & 15:
            t = t.clone(memory_format=torch.contiguous_format)
        return t


def _not_as_saved(t: torch.Tensor, shape, dtype: torch.dtype, device: torch.device) -> None:
    raise RuntimeError(f"a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}, "
                       f"saved was {dtype} {tuple(shape)} on {device}")


def rows_grad(z: torch.Tensor, desc: RowsDesc) -> torch.Tensor:
    """A new tensor for the gradient of rows that lie as ``z``; sets the descriptor's gradient strides."""
    dz = torch.empty_like(z)
    if dz.stride() != z.stride():                        # z overlaps or has gaps: a dense class-last gradient
        dz = class_last_empty(z)
        inner, so, si, sc = _row_strides(dz)
        if desc.inner != inner:                          # the gradient's rows in the logits' (outer, inner) split
            so = si * desc.inner
        desc.grad_outer_stride, desc.grad_inner_stride, desc.grad_class_stride = so, si, sc
    return dz


def _grad_inc(g: Optional[torch.Tensor]):
    """(fp32 tensor, increment per row) of an upstream gradient: one shared value has increment 0."""
    if g is None:
        return None, 0
    if g.dtype != torch.float32:
        g = g.float()
    if g.is_contiguous():
        return g, 1
    if not any(g.stride()):
        return g[(0,) * g.dim()], 0
    return g.contiguous(), 1


def _launch(what: str, fn, dev: torch.device, *args) -> None:
    """Calls a row entry with the device current and its current stream last."""
    index = dev.index
    if index == torch.cuda.current_device():
        st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if st != R4C_OK:
        _check(st, what)


def logp_forward(rows: Rows, target: Optional[torch.Tensor], ignore_index: int, top_k: int, want_stats: bool):
    """(logp or None, entropy, lse, top_logp or None, top_index or None, stats or None)."""
    L, d, z = lib(), rows.desc, rows.z
    shape = rows.shape
    entropy = z.new_empty(shape, dtype=torch.float32)
    lse = torch.empty_like(entropy)
    logp = tl = ti = stats = None
    if target is not None:
        logp = torch.empty_like(entropy)
    if top_k:
        tl = z.new_empty((*shape, top_k), dtype=torch.float32)
        ti = torch.empty_like(tl, dtype=torch.int32)
    if want_stats:
        nb = L.r4c_logp_stats_size(d)
        if nb:
            stats = z.new_empty(nb, dtype=torch.uint8)
    _launch("r4c_logp_fwd", L.r4c_logp_fwd, z.device, d, z.data_ptr(), None if target is None else target.data_ptr(),
            ignore_index, top_k, None if logp is None else logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
            None if tl is None else tl.data_ptr(), None if ti is None else ti.data_ptr(),
            None if stats is None else stats.data_ptr())
    return logp, entropy, lse, tl, ti, stats


def logp_backward(z: torch.Tensor, desc: RowsDesc, target: Optional[torch.Tensor], ignore_index: int,
                  entropy: torch.Tensor, stats: Optional[torch.Tensor], g_logp, g_entropy, g_lse) -> torch.Tensor:
    dz = rows_grad(z, desc)
    (gl, il), (gh, ih), (gs, is_) = _grad_inc(g_logp), _grad_inc(g_entropy), _grad_inc(g_lse)
    _launch("r4c_logp_bwd", lib().r4c_logp_bwd, z.device, desc, z.data_ptr(),
            None if target is None else target.data_ptr(), ignore_index, entropy.data_ptr(),
            None if stats is None else stats.data_ptr(), None if gl is None else gl.data_ptr(), il,
            None if gh is None else gh.data_ptr(), ih, None if gs is None else gs.data_ptr(), is_, dz.data_ptr())
    return dz


def distill_forward(rows: Rows, teacher_logp: torch.Tensor, teacher_index: torch.Tensor, rest: bool,
                    weight: Optional[torch.Tensor], mean: bool):
    """(loss, state): the mean over rows or the rows' own losses, and what the backward needs."""
    L, d, z = lib(), rows.desc, rows.z
    loss = z.new_empty(() if mean else rows.shape, dtype=torch.float32)
    nb = L.r4c_distill_state_size(d)
    state = z.new_empty(nb, dtype=torch.uint8)
    at = loss.data_ptr()
    _launch("r4c_distill_fwd", L.r4c_distill_fwd, z.device, d, z.data_ptr(), teacher_logp.shape[-1],
            teacher_logp.data_ptr(), dtype_code(teacher_logp.dtype), teacher_index.data_ptr(),
            8 * teacher_index.element_size(), rest, None if weight is None else weight.data_ptr(),
            None if mean else at, at if mean else None, state.data_ptr(), nb)
    return loss, state


def distill_backward(z: torch.Tensor, desc: RowsDesc, teacher_logp: torch.Tensor, teacher_index: torch.Tensor,
                     rest: bool, weight: Optional[torch.Tensor], mean: bool, state: torch.Tensor,
                     grad: torch.Tensor) -> torch.Tensor:
    dz = rows_grad(z, desc)
    g, inc = _grad_inc(grad)
    _launch("r4c_distill_bwd", lib().r4c_distill_bwd, z.device, desc, z.data_ptr(), teacher_logp.shape[-1],
            teacher_logp.data_ptr(), dtype_code(teacher_logp.dtype), teacher_index.data_ptr(),
            8 * teacher_index.element_size(), rest, None if weight is None else weight.data_ptr(), mean,
            g.data_ptr(), 0 if mean else inc, state.data_ptr(), dz.data_ptr())
    return dz


# ---------------------------------------------------------------------------
# Activations in 8 bits (r4c_pack8, r4c_unpack8); group normalisation (r4c_gn_*)
# ---------------------------------------------------------------------------
Q8_BLOCK = 32
Q8_FORMATS = {"int8": 0, "e4m3": 1}
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "silu": 3, "gelu": 4}


def q8_buffers(x: torch.Tensor):
    """Empty codes and exponents for x's elements."""
    count = x.numel()
    return x.new_empty(count, dtype=torch.uint8), x.new_empty((count + Q8_BLOCK - 1) // Q8_BLOCK, dtype=torch.uint8)


def pack8(x: torch.Tensor, fmt: int):
    """(codes, exponents) of a dense tensor's elements in memory order."""
    codes, exps = q8_buffers(x)
    _launch("r4c_pack8", lib().r4c_pack8, x.device, x.data_ptr(), codes.shape[0], dtype_code(x.dtype), fmt,
            codes.data_ptr(), exps.data_ptr())
    return codes, exps


def unpack8(codes: torch.Tensor, exps: torch.Tensor, fmt: int, out: torch.Tensor) -> torch.Tensor:
    """Writes the values of the codes into a dense tensor, in its memory order."""
    _launch("r4c_unpack8", lib().r4c_unpack8, out.device, codes.data_ptr(), exps.data_ptr(), out.numel(),
            dtype_code(out.dtype), fmt, out.data_ptr())
    return out


def _up(n: int, unit: int) -> int:
    return (n + unit - 1) // unit * unit


class GnPlan:
    """A descriptor with the sizes of what goes with it: ``stats`` floats that the forward writes for the backward, in
    one allocation with the forward's own workspace (``kept`` floats in all); of the 8 bits the codes' end and the
    whole (``q8_at``, ``q8_bytes``); the backward's workspace."""
    __slots__ = ("desc", "stats", "kept", "ws_at", "fwd_bytes", "bwd_bytes", "q8_at", "q8_bytes")

    def __init__(self, desc: GnDesc):
        L = lib()
        count = desc.samples * desc.inner * desc.channels
        self.desc, self.stats = desc, 2 * desc.samples * desc.groups
        self.fwd_bytes, self.bwd_bytes = L.r4c_gn_workspace_size(desc, 0), L.r4c_gn_workspace_size(desc, 1)
        self.ws_at = _up(4 * self.stats, 256)
        self.kept = (self.ws_at + self.fwd_bytes) // 4 if self.fwd_bytes else self.stats
        self.q8_at = _up(count, 256)
        # (the backward reads exponents in words)
        self.q8_bytes = self.q8_at + _up((count + Q8_BLOCK - 1) // Q8_BLOCK, 4)


@functools.lru_cache(maxsize=512)
def gn_plan(shape: torch.Size, groups: int, dtype: torch.dtype, params_dtype: torch.dtype, eps: float, activation: int,
            slope: float) -> GnPlan:
    """The plan of a call's sizes and types (its kernels are chosen by those alone)."""
    return GnPlan(GnDesc(shape[0], shape[2:].numel(), shape[1], groups, dtype_code(dtype), dtype_code(params_dtype),
                         activation, eps, slope))


def gn_forward(x: torch.Tensor, plan: GnPlan, weight, bias, fmt: Optional[int]):
    """(y, stats, x's 8 bits or None) of a channels-last dense x. Few allocations: each is some microseconds of a call."""
    y = torch.empty_like(x)
    stats = x.new_empty(plan.kept, dtype=torch.float32)
    q8, codes, exps = None, None, None
    if fmt is not None:
        q8 = x.new_empty(plan.q8_bytes, dtype=torch.uint8)
        codes = q8.data_ptr()
        exps = codes + plan.q8_at
    nb, at = plan.fwd_bytes, stats.data_ptr()
    _launch("r4c_gn_fwd", _lib.r4c_gn_fwd, x.device, plan.desc, x.data_ptr(), None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr(), y.data_ptr(), at, fmt or 0, codes, exps,
            at + plan.ws_at if nb else None, nb)
    return y, stats, q8


def gn_backward(dy: torch.Tensor, plan: GnPlan, x, fmt: Optional[int], stats, weight, bias, need_dx: bool,
                need_params: bool):
    """(dx, dweight, dbias); fp32 parameter gradients; x the activation, or with ``fmt`` its 8 bits."""
    dx = torch.empty_like(dy) if need_dx else None
    dw = db = None
    if need_params:
        dw = dy.new_empty((plan.desc.channels,), dtype=torch.float32)
        db = torch.empty_like(dw)
    nb, at = plan.bwd_bytes, x.data_ptr()
    ws = dy.new_empty(nb, dtype=torch.uint8)
    _launch("r4c_gn_bwd", _lib.r4c_gn_bwd, dy.device, plan.desc, dy.data_ptr(), at, fmt or 0,
            None if fmt is None else at + plan.q8_at, stats.data_ptr(),
            None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
            None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
            None if db is None else db.data_ptr(), ws.data_ptr(), nb)
    return dx, dw, db
