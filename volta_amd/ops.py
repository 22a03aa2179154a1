"""Operators of a feed-forward block on device tensors, over the volta_op_* C
ABI (include/volta_ops.h): Linear, GatedFF, RmsNorm and Dropout, forward and
backward, in float32 ("f32"), bfloat16 ("bf16") and float16 ("f16").

An operator object holds the description of its matrices (sizes, types, row
distances); a call takes the matrices themselves, as raw device addresses,
DeviceArrays or anything with data_ptr() (a torch tensor), enqueues its
kernels on `stream` (a hipStream_t as an integer; 0: the default stream, also
where torch's current one is another: pass its cuda_stream) of the current
device and returns.  Outputs, and a workspace of workspace_bytes() where that
is not 0, are the caller's.

A torch tensor's type, shape and strides have to fit the description (rows of
its last dimension, or a flat buffer; as many rows or more), a DeviceArray's
bytes too; nothing is known of a raw address.  What does not fit, and an error
of the library, raises OperatorError with a message.

    op = Linear(rows, inputs, outputs, "bf16", act="gelu")
    op.forward(x, w, y, bias=b, pre=pre, workspace=ws)
    op.backward(dy, x, w, pre=pre, dx=dx, dw=dw, db=db, workspace=ws)
"""
from __future__ import annotations

import ctypes as C

from .abi import ACTIVATIONS

TYPES = {"f32": 0, "bf16": 1, "f16": 2, "e4m3": 3}
ACTS = {"identity": -1, **{k: v for k, v in ACTIVATIONS.items() if k != "softmax"}}
FORWARD, BACKWARD = 0, 1
MASK64 = (1 << 64) - 1


class OperatorError(RuntimeError):
    """A refused call: the library's message, or which matrix does not fit the description."""


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


# What torch tensors may hold a type, by the names of torch's types; what an
# element takes.
_TORCH = {0: ("float32",), 1: ("bfloat16",), 2: ("float16",), 3: ("float8_e4m3fn", "uint8")}
_SIZE = {0: 4, 1: 2, 2: 2, 3: 1}
_NAMES = {v: k for k, v in TYPES.items()}


def _lies(shape, strides, rows, cols, ld) -> bool:
    """Whether a tensor of this shape and these strides holds `rows` rows of
    `cols` elements `ld` apart, or more of them: its last dimension is a row,
    those before it count the rows; one dimension alone is a flat buffer."""
    if rows <= 0:
        return True
    dims = [(n, s) for n, s in zip(shape, strides) if n != 1]
    if any(n == 0 for n, _ in dims):
        return False
    if len(dims) <= 1 and (not dims or dims[0][1] == 1):
        n = dims[0][0] if dims else 1
        if n >= (rows - 1) * ld + cols:
            return True
    if cols != 1:
        if not dims or dims[-1] != (cols, 1):
            return False
        dims.pop()
    if rows == 1:
        return True
    have, apart = 1, ld
    for n, s in reversed(dims):  # rows of rows, each `apart` from the next
        if s != apart:
            return False
        have, apart = have * n, apart * n
    return have >= rows


def _matrix(name, type, rows, cols, ld=0):
    """Returns how the address of matrix `name` of a call is taken: of a raw
    address or of None as it is; of a torch tensor once its type, shape and
    strides fit the description; of a DeviceArray once its bytes do."""
    ld, dtype = ld or cols, None  # dtype: torch's, once a tensor has come by
    shape, nbytes = (rows, cols) if ld == cols else None, rows * cols * _SIZE.get(type, 0)

    def compare(m):
        nonlocal dtype
        if isinstance(m, int):
            return m
        if hasattr(m, "data_ptr"):
            if hasattr(m, "dtype") and hasattr(m, "stride"):
                if str(m.dtype).rpartition(".")[2] not in _TORCH.get(type, ()):
                    raise OperatorError("%s is of %s, the description says %s"
                                        % (name, m.dtype, _NAMES.get(type, type)))
                dtype = m.dtype
                if not _lies(tuple(m.shape), tuple(m.stride()), rows, cols, ld):
                    raise OperatorError("%s has shape %s and strides %s, the description says %d rows of %d, %d apart"
                                        % (name, tuple(m.shape), tuple(m.stride()), rows, cols, ld))
            return m.data_ptr()
        need = ((rows - 1) * ld + cols) * _SIZE.get(type, 0) if rows > 0 else 0
        if getattr(m, "nbytes", need) < need:
            raise OperatorError("%s holds %d bytes, the description says %d" % (name, m.nbytes, need))
        return m.ptr

    # The usual tensor, compared in the fewest steps (a call takes a few
    # microseconds); of a row alone its bytes say as much as its shape.
    def row(m):
        if m is None or m.__class__ is int:
            return m
        try:
            if m.dtype is dtype and m.nbytes == nbytes and m.is_contiguous():
                return m.data_ptr()
        except AttributeError:
            pass
        return compare(m)

    def matrix(m):
        if m is None or m.__class__ is int:
            return m
        try:
            if m.dtype is dtype and m.shape == shape and m.is_contiguous():
                return m.data_ptr()
        except AttributeError:
            pass
        return compare(m)

    return row if rows == 1 else matrix


def _address(m):
    """A workspace's device address; None stays None."""
    if m is None or isinstance(m, int):
        return m
    return m.data_ptr() if hasattr(m, "data_ptr") else m.ptr


def _bytes(m) -> int:
    """Bytes of a workspace the caller holds; a raw address is taken at its word."""
    if m is None:
        return 0
    if isinstance(m, int):
        return (1 << 63) - 1
    return int(m.nbytes)


class _Operator:
    def __init__(self, desc, name, lib=None):
        from volta_amd import load_hip

        self.lib = bind((lib or load_hip()).lib)
        self.desc = desc
        self._d = C.byref(desc)
        self._name = name

    def _fn(self, call):
        return getattr(self.lib, "volta_op_%s_%s" % (self._name, call))

    def _refused(self):
        return OperatorError(self.lib.volta_rt_last_error().decode())

    def workspace_bytes(self, backward: bool = False) -> int:
        """Bytes of workspace that a forward or backward call needs."""
        n = self._fn("workspace")(self._d, BACKWARD if backward else FORWARD)
        if n < 0:
            raise self._refused()
        return int(n)


class Linear(_Operator):
    """y = act(x W + bias) + residual, and its gradients.  ld_*: distance
    between a matrix's rows in elements (0: packed)."""

    def __init__(self, rows, inputs, outputs, dtype="f32", act="identity", ld_x=0, ld_w=0, ld_y=0, ld_residual=0,
                 ld_pre=0, ld_dx=0, ld_dw=0, lib=None):
        t = TYPES[dtype]
        super().__init__(LinearDesc(t, ACTS[act], rows, inputs, outputs, ld_x, ld_w, ld_y, ld_residual, ld_pre, ld_dx,
                                    ld_dw), "linear", lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")
        x, w = _matrix("x", t, rows, inputs, ld_x), _matrix("w", t, inputs, outputs, ld_w)
        pre = _matrix("pre", t, rows, outputs, ld_pre)
        self._of_forward = (x, w, _matrix("bias", t, 1, outputs), _matrix("residual", t, rows, outputs, ld_residual),
                            _matrix("y", t, rows, outputs, ld_y), pre)
        self._of_backward = (_matrix("dy", t, rows, outputs, ld_y), x, w, pre, _matrix("dx", t, rows, inputs, ld_dx),
                             _matrix("dw", t, inputs, outputs, ld_dw), _matrix("db", t, 1, outputs))

    def forward(self, x, w, y, bias=None, residual=None, pre=None, workspace=None, stream=0):
        ax, aw, ab, ar, ay, ap = self._of_forward
        if self._forward(self._d, ax(x), aw(w), ab(bias), ar(residual), ay(y), ap(pre), _address(workspace),
                         _bytes(workspace), stream):
            raise self._refused()

    def backward(self, dy, x, w, pre=None, dx=None, dw=None, db=None, workspace=None, stream=0):
        ay, ax, aw, ap, adx, adw, adb = self._of_backward
        if self._backward(self._d, ay(dy), ax(x), aw(w), ap(pre), adx(dx), adw(dw), adb(db),
                          _address(workspace), _bytes(workspace), stream):
            raise self._refused()


class GatedFF(_Operator):
    """h = act(x Wg + bg) * (x Wu + bu), and its gradients."""

    def __init__(self, rows, inputs, hidden, dtype="f32", act="silu", ld_x=0, ld_w=0, ld_h=0, ld_pre=0, ld_dx=0,
                 ld_dw=0, lib=None):
        t = TYPES[dtype]
        super().__init__(GatedDesc(t, ACTS[act], rows, inputs, hidden, ld_x, ld_w, ld_h, ld_pre, ld_dx, ld_dw), "gated",
                         lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")
        x = _matrix("x", t, rows, inputs, ld_x)
        w = [_matrix(n, t, inputs, hidden, ld_w) for n in ("w_gate", "w_up")]
        pre = [_matrix(n, t, rows, hidden, ld_pre) for n in ("gate", "up")]
        self._of_forward = (x, *w, _matrix("b_gate", t, 1, hidden), _matrix("b_up", t, 1, hidden),
                            _matrix("h", t, rows, hidden, ld_h), *pre)
        self._of_backward = (_matrix("dh", t, rows, hidden, ld_h), x, *w, *pre, _matrix("dx", t, rows, inputs, ld_dx),
                             _matrix("dw_gate", t, inputs, hidden, ld_dw), _matrix("dw_up", t, inputs, hidden, ld_dw),
                             _matrix("db_gate", t, 1, hidden), _matrix("db_up", t, 1, hidden))

    def forward(self, x, w_gate, w_up, h, b_gate=None, b_up=None, gate=None, up=None, workspace=None, stream=0):
        ax, awg, awu, abg, abu, ah, ag, au = self._of_forward
        if self._forward(self._d, ax(x), awg(w_gate), awu(w_up), abg(b_gate), abu(b_up), ah(h), ag(gate),
                         au(up), _address(workspace), _bytes(workspace), stream):
            raise self._refused()

    def backward(self, dh, x, w_gate, w_up, gate, up, dx=None, dw_gate=None, dw_up=None, db_gate=None, db_up=None,
                 workspace=None, stream=0):
        ah, ax, awg, awu, ag, au, adx, adg, adu, abg, abu = self._of_backward
        if self._backward(self._d, ah(dh), ax(x), awg(w_gate), awu(w_up), ag(gate), au(up), adx(dx),
                          adg(dw_gate), adu(dw_up), abg(db_gate), abu(db_up), _address(workspace),
                          _bytes(workspace), stream):
            raise self._refused()


class RmsNorm(_Operator):
    """s = x + residual; y = s / sqrt(mean(s^2) + eps) * weight, in the
    inputs' type (out="same") or as e4m3 codes with a scale for each row
    (out="e4m3") or for each 128 columns (group=128); and its gradients."""

    def __init__(self, rows, cols, dtype="f32", eps=1e-6, out="same", group=0, ld_x=0, ld_residual=0, ld_sum=0,
                 ld_y=0, ld_dx=0, lib=None):
        t, to = TYPES[dtype], TYPES[dtype if out == "same" else out]
        super().__init__(RmsNormDesc(t, to, rows, cols, eps, group, ld_x, ld_residual, ld_sum, ld_y, ld_dx), "rms_norm",
                         lib)
        self._forward, self._backward = self._fn("forward"), self._fn("backward")
        weight, rstd = _matrix("weight", t, 1, cols), _matrix("rstd", TYPES["f32"], 1, rows)
        scales = _matrix("scales", TYPES["f32"], rows, -(-cols // group) if group > 0 else 1)
        self._of_forward = (_matrix("x", t, rows, cols, ld_x), _matrix("residual", t, rows, cols, ld_residual), weight,
                            _matrix("y", to, rows, cols, ld_y), _matrix("sum", t, rows, cols, ld_sum), rstd, scales)
        self._of_backward = (_matrix("dy", t, rows, cols, ld_y), _matrix("s", t, rows, cols, ld_x), rstd, weight,
                             _matrix("dsum", t, rows, cols, ld_sum), _matrix("dx", t, rows, cols, ld_dx),
                             _matrix("dweight", t, 1, cols))

    def forward(self, x, y, weight=None, residual=None, sum=None, rstd=None, scales=None, stream=0):
        ax, ar, aw, ay, asum, arstd, ascales = self._of_forward
        if self._forward(self._d, ax(x), ar(residual), aw(weight), ay(y), asum(sum), arstd(rstd),
                         ascales(scales), stream):
            raise self._refused()

    def backward(self, dy, s, rstd, dx=None, weight=None, dsum=None, dweight=None, workspace=None, stream=0):
        ay, asum, arstd, aw, ads, adx, adw = self._of_backward
        if self._backward(self._d, ay(dy), asum(s), arstd(rstd), aw(weight), ads(dsum), adx(dx), adw(dweight),
                          _address(workspace), _bytes(workspace), stream):
            raise self._refused()


class Dropout(_Operator):
    """y = residual + x keep / (1 - p); the mask is drawn from (seed, offset),
    so the backward pass is the same call on dy."""

    def __init__(self, rows, cols, dtype="f32", p=0.1, ld_x=0, ld_residual=0, ld_y=0, lib=None):
        t = TYPES[dtype]
        super().__init__(DropoutDesc(t, p, rows, cols, ld_x, ld_residual, ld_y), "dropout", lib)
        self._forward = self._fn("forward")
        self._of_forward = (_matrix("x", t, rows, cols, ld_x), _matrix("residual", t, rows, cols, ld_residual),
                            _matrix("y", t, rows, cols, ld_y))
        self._of_backward = (_matrix("dy", t, rows, cols, ld_x), _matrix("dx", t, rows, cols, ld_y))

    def forward(self, x, y, residual=None, seed=0, offset=0, stream=0):
        ax, ar, ay = self._of_forward
        if self._forward(self._d, ax(x), ar(residual), ay(y), seed & MASK64, offset & MASK64, stream):
            raise self._refused()

    def backward(self, dy, dx, seed=0, offset=0, stream=0):
        """The gradient of x (the residual's is dy)."""
        ay, ax = self._of_backward
        if self._forward(self._d, ay(dy), None, ax(dx), seed & MASK64, offset & MASK64, stream):
            raise self._refused()

    def workspace_bytes(self, backward: bool = False) -> int:
        return 0
