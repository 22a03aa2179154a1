"""Which products of a layer a call looks at (include/volta_ops.h): those that
it runs.  Without a GPU: the calls are refused on the host, for the products
they run or, where those are fine, for the lack of a device or of memory."""
from __future__ import annotations

import os

import pytest

from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")

# far enough apart for the largest matrix below
A = [(i + 1) << 46 for i in range(12)]


def said(call, **kw):
    with pytest.raises(ops.OperatorError) as e:
        call(**kw)
    return str(e.value)


def test_rows_too_many_for_dx_alone():
    """2^30 rows are too many tiles of dx; dW and the biases' gradients are sums over them."""
    lin = ops.Linear(1 << 30, 64, 64, "bf16")
    assert "too many" in said(lin.backward, dy=A[0], x=A[1], w=A[2], dx=A[3], workspace=A[8])
    assert "too many" in said(lin.backward, dy=A[0], x=A[1], w=A[2], dx=A[3], dw=A[4], workspace=A[8])
    for kw in ({"dw": A[4]}, {"db": A[5]}, {"dw": A[4], "db": A[5]}):
        assert "too many" not in said(lin.backward, dy=A[0], x=A[1], w=A[2], workspace=A[8], **kw)
    gat = ops.GatedFF(1 << 30, 64, 64, "bf16")
    args = dict(zip(("dh", "x", "w_gate", "w_up", "gate", "up"), A))
    assert "too many" in said(gat.backward, dx=A[6], workspace=A[11], **args)
    for kw in ({"dw_gate": A[7], "dw_up": A[8]}, {"db_gate": A[9]}, {"db_up": A[10]}):
        assert "too many" not in said(gat.backward, workspace=A[11], **kw, **args)


def test_weights_too_many_for_dw_alone():
    """2^19 by 2^19 weights are too many tiles of dW; a row through them is not."""
    n = 1 << 19
    lin, gat = ops.Linear(1, n, n, "bf16"), ops.GatedFF(1, n, n, "bf16")
    assert "too many" in said(lin.backward, dy=A[0], x=A[1], w=A[2], dw=A[3], workspace=A[8])
    assert "too many" not in said(lin.backward, dy=A[0], x=A[1], w=A[2], dx=A[3], workspace=A[8])
    assert "too many" not in said(lin.forward, x=A[0], w=A[1], y=A[2], workspace=A[8])
    args = dict(zip(("dh", "x", "w_gate", "w_up", "gate", "up"), A))
    assert "too many" in said(gat.backward, dw_gate=A[6], dw_up=A[7], workspace=A[11], **args)
    assert "too many" not in said(gat.backward, dx=A[6], workspace=A[11], **args)


def test_a_workspace_speaks_for_every_gradient():
    for op in (ops.Linear(1 << 30, 64, 64, "bf16"), ops.Linear(1, 1 << 19, 1 << 19, "bf16"),
               ops.GatedFF(1 << 30, 64, 64, "f16")):
        assert "too many" in said(op.workspace_bytes, backward=True)
    assert ops.Linear(1, 1 << 19, 1 << 19, "bf16").workspace_bytes() >= 0


def test_a_refusal_says_what_the_call_takes():
    class Short:
        ptr, nbytes = A[8], 0

    lin = ops.Linear(1 << 30, 64, 64, "bf16")
    text = said(lin.backward, dy=A[0], x=A[1], w=A[2], dw=A[4], workspace=Short)
    assert "holds 0 bytes" in text and int(text.split("needed are ")[1]) > 0
