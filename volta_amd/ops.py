"""Operators of a feed-forward block on device tensors, over the volta_op_* C
ABI (include/volta_ops.h): Linear, GatedFF, RmsNorm and Dropout, forward and
backward, in float32 ("f32"), bfloat16 ("bf16") and float16 ("f16").

An operator object holds the description of its matrices (sizes, types, row
distances); a call takes the matrices themselves, as raw device addresses,
DeviceArrays or anything with data_ptr() (a torch tensor), enqueues its
kernels on `stream` (a hipStream_t as an integer; 0: the default stream) of
the current device and returns.  Outputs, and a workspace of
workspace_bytes() where that is not 0, are the caller's.  An error of the
library raises OperatorError with its message.

    op = Linear(rows, inputs, outputs, "bf16", act="gelu")
    op.forward(x, w, y, bias=b, pre=pre, workspace=ws)
    op.backward(dy, x, w, pre=pre, dx=dx, dw=dw, db=db, workspace=ws)
"""
from __future__ import annotations

import ctypes as C
from operator import attrgetter

from .abi import ACTIVATIONS

TYPES = {"f32": 0, "bf16": 1, "f16": 2, "e4m3": 3}
ACTS = {"identity": -1, **{k: v for k, v in ACTIVATIONS.items() if k != "softmax"}}
FORWARD, BACKWARD = 0, 1
MASK64 = (1 << 64) - 1


class OperatorError(RuntimeError):
    """The library's message."""


class LinearDesc(C.Structure):
    _fields_ = [("type", C.c_int32), ("act", C.c_int32)] + [
        (n, C.c_int64) for n in ("rows", "inputs", "outputs", "ld_x", "ld_w", "ld_y", "ld_residual", "ld_pre", "ld_dx",
                                 "ld_dw")]


class GatedDesc(C.Structure):
    _fields_ = [("type", C.c_int32), ("act", C.c_int32)] + [
        (n, C.c_int64) for n in ("rows", "inputs", "hidden", "ld_x", "ld_w", "ld_h", "ld_pre", "ld_dx", "ld_dw")]


class RmsNormDesc(C.Structure):
    _fields_ = [("type", C.c_int32), ("out_type", C.c_int32), ("rows", C.c_int64), ("cols", C.c_int64),
                ("eps", C.c_float), ("group", C.c_int32)] + [
        (n, C.c_int64) for n in ("ld_x", "ld_residual", "ld_sum", "ld_y", "ld_dx")]


class DropoutDesc(C.Structure):
    _fields_ = [("type", C.c_int32), ("p", C.c_double)] + [
        (n, C.c_int64) for n in ("rows", "cols", "ld_x", "ld_residual", "ld_y")]


_P, _N = C.c_void_p, C.c_int64

SIGNATURES = {
    "volta_op_linear_workspace": (_N, [C.POINTER(LinearDesc), C.c_int32]),
    "volta_op_linear_forward": (C.c_int32, [C.POINTER(LinearDesc)] + [_P] * 7 + [_N, _P]),
    "volta_op_linear_backward": (C.c_int32, [C.POINTER(LinearDesc)] + [_P] * 8 + [_N, _P]),
    "volta_op_gated_workspace": (_N, [C.POINTER(GatedDesc), C.c_int32]),
    "volta_op_gated_forward": (C.c_int32, [C.POINTER(GatedDesc)] + [_P] * 9 + [_N, _P]),
    "volta_op_gated_backward": (C.c_int32, [C.POINTER(GatedDesc)] + [_P] * 12 + [_N, _P]),
    "volta_op_rms_norm_workspace": (_N, [C.POINTER(RmsNormDesc), C.c_int32]),
    "volta_op_rms_norm_forward": (C.c_int32, [C.POINTER(RmsNormDesc)] + [_P] * 8),
    "volta_op_rms_norm_backward": (C.c_int32, [C.POINTER(RmsNormDesc)] + [_P] * 8 + [_N, _P]),
    "volta_op_dropout_forward": (C.c_int32, [C.POINTER(DropoutDesc), _P, _P, _P, C.c_uint64, C.c_uint64, _P]),
}


def bind(cdll: C.CDLL) -> C.CDLL:
    """Declare the volta_op_* signatures on a loaded library (once)."""
    if getattr(cdll, "_volta_ops_bound", False):
        return cdll
    cdll._volta_ops_bound = True
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(cdll, name)
        fn.restype = res
        fn.argtypes = args
    cdll.volta_rt_last_error.restype = C.c_char_p
    return cdll


_READERS: dict = {}


def _reader(t):
    """How a matrix of type t gives its device address."""
    read = int if issubclass(t, int) else t.data_ptr if hasattr(t, "data_ptr") else attrgetter("ptr")
    _READERS[t] = read
    return read


def _address(m):
    """A matrix's device address; None stays None."""
    if m is None:
        return None
    t = type(m)
    return (_READERS.get(t) or _reader(t))(m)


def _bytes(m) -> int:
    """Bytes of a workspace the caller holds; a raw address is taken at its word."""
    if m is None:
        return 0
    if isinstance(m, int):
        return (1 << 63) - 1
    if hasattr(m, "ptr"):
        return int(m.nbytes)
    return int(m.numel() * m.element_size())


class _Operator:
    def __init__(self, desc, name, lib=None):
        from volta_amd import load_hip

        self.lib = bind((lib or load_hip()).lib)
        self.desc = desc
        self._d = C.byref(desc)
        self._name = name

    def _fn(self, call):
        return getattr(self.lib, "volta_op_%s_%s" % (self._name, call))

    def _check(self, rc):
        if rc != 0:
            raise OperatorError(self.lib.volta_rt_last_error().decode())

    def workspace_bytes(self, backward: bool = False) -> int:
        """Bytes of workspace that a forward or backward call needs."""
        n = self._fn("workspace")(self._d, BACKWARD if backward else FORWARD)
        if n < 0:
            raise OperatorError(self.lib.volta_rt_last_error().decode())
        return int(n)


class Linear(_Operator):
    """y = act(x W + bias) + residual, and its gradients.  ld_*: distance
    between a matrix's rows in elements (0: packed)."""

    def __init__(self, rows, inputs, outputs, dtype="f32", act="identity", ld_x=0, ld_w=0, ld_y=0, ld_residual=0,
                 ld_pre=0, ld_dx=0, ld_dw=0, lib=None):
        super().__init__(LinearDesc(TYPES[dtype], ACTS[act], rows, inputs, outputs, ld_x, ld_w, ld_y, ld_residual,
                                    ld_pre, ld_dx, ld_dw), "linear", lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")

    def forward(self, x, w, y, bias=None, residual=None, pre=None, workspace=None, stream=0):
        a = _address
        self._check(self._forward(self._d, a(x), a(w), a(bias), a(residual), a(y), a(pre), a(workspace),
                                  _bytes(workspace), stream))

    def backward(self, dy, x, w, pre=None, dx=None, dw=None, db=None, workspace=None, stream=0):
        a = _address
        self._check(self._backward(self._d, a(dy), a(x), a(w), a(pre), a(dx), a(dw), a(db), a(workspace),
                                   _bytes(workspace), stream))


class GatedFF(_Operator):
    """h = act(x Wg + bg) * (x Wu + bu), and its gradients."""

    def __init__(self, rows, inputs, hidden, dtype="f32", act="silu", ld_x=0, ld_w=0, ld_h=0, ld_pre=0, ld_dx=0,
                 ld_dw=0, lib=None):
        super().__init__(GatedDesc(TYPES[dtype], ACTS[act], rows, inputs, hidden, ld_x, ld_w, ld_h, ld_pre, ld_dx,
                                   ld_dw), "gated", lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")

    def forward(self, x, w_gate, w_up, h, b_gate=None, b_up=None, gate=None, up=None, workspace=None, stream=0):
        a = _address
        self._check(self._forward(self._d, a(x), a(w_gate), a(w_up), a(b_gate), a(b_up), a(h), a(gate), a(up),
                                  a(workspace), _bytes(workspace), stream))

    def backward(self, dh, x, w_gate, w_up, gate, up, dx=None, dw_gate=None, dw_up=None, db_gate=None, db_up=None,
                 workspace=None, stream=0):
        a = _address
        self._check(self._backward(self._d, a(dh), a(x), a(w_gate), a(w_up), a(gate), a(up), a(dx), a(dw_gate),
                                   a(dw_up), a(db_gate), a(db_up), a(workspace), _bytes(workspace), stream))


class RmsNorm(_Operator):
    """s = x + residual; y = s / sqrt(mean(s^2) + eps) * weight, in the
    inputs' type (out="same") or as e4m3 codes with a scale for each row
    (out="e4m3") or for each 128 columns (group=128); and its gradients."""

    def __init__(self, rows, cols, dtype="f32", eps=1e-6, out="same", group=0, ld_x=0, ld_residual=0, ld_sum=0,
                 ld_y=0, ld_dx=0, lib=None):
        super().__init__(RmsNormDesc(TYPES[dtype], TYPES[dtype if out == "same" else out], rows, cols, eps, group, ld_x,
                                     ld_residual, ld_sum, ld_y, ld_dx), "rms_norm", lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")

    def forward(self, x, y, weight=None, residual=None, sum=None, rstd=None, scales=None, stream=0):
        a = _address
        self._check(self._forward(self._d, a(x), a(residual), a(weight), a(y), a(sum), a(rstd), a(scales), stream))

    def backward(self, dy, s, rstd, dx=None, weight=None, dsum=None, dweight=None, workspace=None, stream=0):
        a = _address
        self._check(self._backward(self._d, a(dy), a(s), a(rstd), a(weight), a(dsum), a(dx), a(dweight), a(workspace),
                                   _bytes(workspace), stream))


class Dropout(_Operator):
    """y = residual + x keep / (1 - p); the mask is drawn from (seed, offset),
    so the backward pass is the same call on dy."""

    def __init__(self, rows, cols, dtype="f32", p=0.1, ld_x=0, ld_residual=0, ld_y=0, lib=None):
        super().__init__(DropoutDesc(TYPES[dtype], p, rows, cols, ld_x, ld_residual, ld_y), "dropout", lib)
        self._forward = self._fn("forward")

    def forward(self, x, y, residual=None, seed=0, offset=0, stream=0):
        a = _address
        self._check(self._forward(self._d, a(x), a(residual), a(y), seed & MASK64, offset & MASK64, stream))

    def backward(self, dy, dx, seed=0, offset=0, stream=0):
        """The gradient of x (the residual's is dy)."""
        self.forward(dy, dx, seed=seed, offset=offset, stream=stream)

    def workspace_bytes(self, backward: bool = False) -> int:
        return 0
