"""Calls of no rows with the tensors that a program then has (volta_amd.ops),
without a GPU: they are not refused for their shapes."""
from __future__ import annotations

import os

import pytest

from tests.test_ops_matrices import Tensor
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def tensor(type, *shape, at=0):
    t = Tensor(type, shape, at=(at + 1) << 32)
    if 0 in shape:
        t.at = 0  # what torch has for one
    return t


def takes(call, *args, **kw):
    """The call is not refused for its matrices (without a device it is for that)."""
    try:
        call(*args, **kw)
    except ops.OperatorError as e:
        assert "the description says" not in str(e) and "NULL" not in str(e), str(e)


def test_no_rows():
    w, half, f32 = tensor("bfloat16", 64, 100), "bfloat16", "float32"
    x, labels = tensor(half, 0, 64, at=1), tensor("int32", 0, at=2)
    loss, lse, dloss = (tensor(f32, 0, at=3 + i) for i in range(3))
    op = ops.CrossEntropy(0, 64, 100, "bf16")
    for _ in range(2):  # the second call compares by what the first one has seen
        takes(op.forward, x, w, labels, loss, lse=lse)
        takes(op.backward, x, w, labels, lse, dloss, dx=tensor(half, 0, 64, at=6), workspace=1 << 40)
        takes(op.backward, x, w, labels, lse, dloss, dx=tensor(half, 0, 64, at=6), dw=tensor(half, 64, 100, at=7),
              workspace=1 << 40)
    norm = ops.RmsNorm(0, 64, "bf16")
    for _ in range(2):
        takes(norm.forward, x, tensor(half, 0, 64, at=8), rstd=tensor(f32, 0, at=9))
        takes(norm.backward, x, x, tensor(f32, 0, at=9), dx=tensor(half, 0, 64, at=8))
    for by, y, scales in (("rows", (0, 64), (0, 1)), ("blocks", (64, 0), (1, 0))):
        codes = ops.Quantize(0, 64, "bf16", by=by)
        for _ in range(2):
            takes(codes.forward, x, tensor("float8_e4m3fn", *y, at=10), tensor(f32, *scales, at=11))
    dy, dx = tensor(half, 0, 100, at=12), tensor(half, 0, 64, at=13)
    takes(ops.Linear(0, 64, 100, "bf16").backward, dy, x, w, dx=dx, workspace=1 << 40)
    takes(ops.GatedFF(0, 64, 100, "bf16").backward, dy, x, w, w, dy, dy, dx=dx, workspace=1 << 40)
    layer = ops.Linear8(0, 64, 100)
    takes(layer.forward, tensor("uint8", 0, 64), tensor(f32, 0, 1), tensor("uint8", 100, 64), tensor(f32, 1, 1),
          tensor(half, 0, 100))


def test_other_types_and_missing_rows_are_refused_still():
    op = ops.CrossEntropy(0, 64, 100, "bf16")
    with pytest.raises(ops.OperatorError, match="labels is of torch.int64"):
        op.forward(tensor("bfloat16", 0, 64), tensor("bfloat16", 64, 100), tensor("int64", 0), tensor("float32", 0))
    op = ops.CrossEntropy(3, 64, 100, "bf16")
    with pytest.raises(ops.OperatorError, match="labels has shape"):
        op.forward(tensor("bfloat16", 3, 64), tensor("bfloat16", 64, 100), tensor("int32", 0), tensor("float32", 3))
