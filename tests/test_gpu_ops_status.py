"""The operators (include/volta_ops.h) in a program whose own HIP call failed
before: a call's result is its own launches', and the program's error is still
there afterwards."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests.ops_ref import Mat
from tests.test_gpu_ops import EPS, Block, Space, draws
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return load_hip()


@pytest.fixture
def failed_call(lib):
    """Makes a HIP call fail on the host, as a program does that tries a device
    too many; returns how its error is read."""
    hip = lib.lib
    hip.hipSetDevice.restype, hip.hipSetDevice.argtypes = C.c_int, [C.c_int]
    hip.hipPeekAtLastError.restype = hip.hipGetLastError.restype = C.c_int

    def fail():
        rc = hip.hipSetDevice(-1)
        assert rc != 0 and hip.hipPeekAtLastError() == rc
        return rc

    yield fail
    hip.hipGetLastError()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_a_block_after_a_failed_call(lib, failed_call, t):
    """Norm, gated and linear layer and dropout, forward and backward, in one
    launch and in several: every output as without the failed call."""
    # 1600 x 1001 x 1501: operands laid out anew; 5 x 2048 x 4096: sums split
    # over blocks; 70 rows: strips' sums added by a launch of their own
    for M, D, H in ((70, 96, 200), (5, 2048, 4096), (1600, 1001, 1501)):
        print(t, M, D, H, flush=True)
        b = Block(lib, t, M, D, H)
        b.run()
        want = b.bits()
        for k in Block.OUT:
            m = b.m[k]
            lib.lib.volta_hip_copy(m.dev.ptr, m.before.ctypes.data, m.before.nbytes, 1)
        rc = failed_call()
        b.run()
        assert lib.lib.hipPeekAtLastError() == rc
        lib.lib.hipGetLastError()
        assert all(np.array_equal(v, want[k]) for k, v in b.bits().items())


def test_wide_rows_and_biases_after_a_failed_call(lib, failed_call):
    """The norm of rows that no block holds, and sums of biases' gradients."""
    rng = np.random.default_rng(2)
    M, D = 40, 34001
    x, dy = Mat(lib, "bf16", M, D, draws(rng, "bf16", M, D)), Mat(lib, "bf16", M, D, draws(rng, "bf16", M, D))
    norm, lin = ops.RmsNorm(M, D, "bf16", EPS), ops.Linear(M, 16, D, "bf16", act="gelu")
    ws, wl = Space(lib, norm, True), Space(lib, lin, True)
    got = []
    for fail in (False, True):
        y, r, dx, dw = Mat(lib, "bf16", M, D), Mat(lib, "f32", 1, M), Mat(lib, "bf16", M, D), Mat(lib, "bf16", 1, D)
        db = Mat(lib, "bf16", 1, D)
        if fail:
            failed_call()
        norm.forward(x, y, rstd=r)
        norm.backward(dy, x, r, dx=dx, dweight=dw, workspace=ws)
        lin.backward(dy, None, None, pre=x, db=db, workspace=wl)
        lib.lib.hipGetLastError()
        got.append([v.bits() for v in (y, r, dx, dw, db)])
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_a_refusal_leaves_no_error_behind(lib):
    """What a call's own lookups say is in its message alone."""
    hip = lib.lib
    hip.hipPeekAtLastError.restype = hip.hipGetLastError.restype = C.c_int
    hip.hipGetLastError()
    host = np.zeros(64, np.float32)
    y, op = Mat(lib, "f32", 4, 8), ops.Dropout(4, 8)
    with pytest.raises(ops.OperatorError):
        op.forward(host.ctypes.data, y)
    assert hip.hipPeekAtLastError() == 0
    x = Mat(lib, "f32", 4, 8, np.ones((4, 8)))
    op.forward(x, y)
    assert hip.hipPeekAtLastError() == 0 and y.get().any()
