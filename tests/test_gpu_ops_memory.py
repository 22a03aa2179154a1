"""Matrices that end behind their memory are refused on the host
(include/volta_ops.h), whichever argument they are."""
from __future__ import annotations

import ctypes as C

import pytest

from tests.ops_ref import Mat
from tests.test_gpu_ops import EPS
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def _range(lib, p):
    """The allocation at p as the runtime gives it: its first byte and its size."""
    fn = lib.lib.hipMemGetAddressRange
    fn.restype, fn.argtypes = C.c_int, [C.POINTER(C.c_void_p), C.POINTER(C.c_size_t), C.c_void_p]
    base, size = C.c_void_p(), C.c_size_t()
    assert fn(C.byref(base), C.byref(size), p) == 0
    return base.value, size.value


# 2^30 rows of 2^20 elements: 2 PB in bf16, more than any run of allocations side by side
ROWS, COLS = 1 << 30, 1 << 20


def test_the_runtime_knows_allocations_ends(lib):
    for n in (64, 4096, 1 << 20, 5 << 20):
        m = Mat(lib, "f32", 1, n // 4)
        base, size = _range(lib, m.ptr + n // 2)
        assert base <= m.ptr and n <= base + size - m.ptr < 1 << 40


def test_short_matrices_refused(lib):
    small = [Mat(lib, "bf16", 4, 64) for _ in range(2)]
    for m in small:
        base, size = _range(lib, m.ptr)
        assert base + size - m.ptr < ROWS  # or the runtime would not refuse what follows
    a = small[0].ptr
    norm, drop = ops.RmsNorm(ROWS, COLS, "bf16", EPS), ops.Dropout(ROWS, COLS, "bf16")

    def refused(name, call):
        with pytest.raises(ops.OperatorError) as e:
            call()
        assert str(e.value).split(": ")[1].startswith(name + " ends "), str(e.value)

    far = 1 << 56  # an address apart from everything: looked up after the short one
    refused("x", lambda: norm.forward(a, far))
    refused("x", lambda: drop.forward(a, far))
    refused("dy", lambda: norm.backward(a, far, 2 * far, dx=3 * far))
    # a short output beside whole inputs below it
    x, w, y = sorted((Mat(lib, "bf16", 64, 64) for _ in range(3)), key=lambda m: m.ptr)
    one = ops.Linear(4, 64, 64, "bf16", ld_y=1 << 21)
    assert one.workspace_bytes() == 0 and _range(lib, y.ptr)[1] < 1 << 21
    if _followed(lib, y.ptr):
        pytest.skip("memory follows the short output's")
    refused("y", lambda: one.forward(x.ptr, w.ptr, y.ptr))
    assert all(m.untouched() for m in small + [x, w, y])


def _followed(lib, p):
    """Whether other memory lies directly behind p's allocation."""
    base, size = _range(lib, p)
    out = (C.c_char * 256)()
    lib.lib.hipPointerGetAttributes.restype = C.c_int
    rc = lib.lib.hipPointerGetAttributes(out, C.c_void_p(base + size))
    kind = int.from_bytes(bytes(out[:4]), "little")
    lib.lib.hipGetLastError()
    return rc == 0 and kind != 0
