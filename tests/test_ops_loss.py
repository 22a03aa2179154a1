"""The loss of an output layer (include/volta_ops.h, volta_amd.ops.CrossEntropy)
without a GPU: what is refused, with which message, and what is planned."""
from __future__ import annotations

import os
import random

import pytest

from tests.test_ops import A, refused
from tests.test_ops_matrices import Tensor
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def test_descriptions_refused():
    for f, text in [(lambda: ops.CrossEntropy(-1, 4, 4), "rows is -1"), (lambda: ops.CrossEntropy(4, 0, 4), "inputs is 0"),
                    (lambda: ops.CrossEntropy(4, 4, 0), "classes is 0"),
                    (lambda: ops.CrossEntropy(4, 4, (1 << 21) + 1), "classes is"),
                    (lambda: ops.CrossEntropy(4, 8, 4, ld_x=7), "ld_x is 7"),
                    (lambda: ops.CrossEntropy(4, 8, 4, ld_w=3), "ld_w is 3"),
                    (lambda: ops.CrossEntropy(4, 8, 4, ld_dx=7), "ld_dx is 7"),
                    (lambda: ops.CrossEntropy(4, 8, 4, ld_dw=(1 << 21) + 1), "ld_dw is")]:
        for backward in (False, True):
            refused(lambda: f().workspace_bytes(backward=backward), text)
    op = ops.CrossEntropy(4, 4, 4)
    op.desc.type = 3
    refused(op.workspace_bytes, "type is 3")


def test_calls_refused():
    op = ops.CrossEntropy(4, 8, 16)
    W = A[12]
    refused(lambda: op.forward(A[0], A[1], A[2], None, workspace=W), "loss and lse are both NULL")
    refused(lambda: op.forward(None, A[1], A[2], A[3], workspace=W), "x is NULL")
    refused(lambda: op.forward(A[0], None, A[2], A[3], workspace=W), "w is NULL")
    refused(lambda: op.forward(A[0], A[1], None, A[3], workspace=W), "labels is NULL")
    refused(lambda: op.forward(A[0], A[1], A[2] + 2, A[3], workspace=W), "labels is not aligned")
    refused(lambda: op.forward(A[0], A[1], A[2], A[3], lse=A[3], workspace=W), "loss and lse overlap")
    refused(lambda: op.forward(A[0], A[1], A[2], A[0], workspace=W), "x and loss overlap")
    refused(lambda: op.forward(A[0], A[1], A[2], A[3]), "workspace holds 0")
    back = (A[0], A[1], A[2], A[3], A[4])
    refused(lambda: op.backward(*back, workspace=W), "all NULL")
    for i, name in enumerate(("x", "w", "labels", "lse", "dloss")):
        args = list(back)
        args[i] = None
        refused(lambda: op.backward(*args, dx=A[5], workspace=W), name + " is NULL")
    refused(lambda: op.backward(*back, dx=A[0], workspace=W), "x and dx overlap")
    refused(lambda: op.backward(*back, dw=A[1], workspace=W), "w and dw overlap")
    refused(lambda: op.backward(*back, dx=A[5], db=A[5], workspace=W), "dx and db overlap")
    refused(lambda: op.backward(*back, dx=A[5], workspace=A[5] + 64), "overlaps the workspace")
    refused(lambda: op.backward(*back, dx=A[5]), "workspace holds 0")


def test_workspace_keeps_a_piece_of_the_gradient():
    """Far below all of dz, and the same from the sizes alone."""
    op = ops.CrossEntropy(8192, 4096, 131072, "bf16")
    n = op.workspace_bytes(backward=True)
    assert (1 << 28) - (1 << 23) < n < 600 << 20 and n == op.workspace_bytes(backward=True)
    assert op.workspace_bytes() < 65 << 20
    assert ops.CrossEntropy(1, 4096, 32768, "bf16").workspace_bytes() < 1 << 20


def test_every_matrix_is_compared():
    M, K, C = 4, 16, 24
    op = ops.CrossEntropy(M, K, C, "bf16")
    shapes = {"x": (M, K), "w": (K, C), "bias": (C,), "labels": (M,), "loss": (M,), "lse": (M,), "dloss": (M,),
              "dx": (M, K), "dw": (K, C), "db": (C,)}
    types = {"labels": "int32", "loss": "float32", "lse": "float32", "dloss": "float32"}
    for call, names in ((op.forward, "x w bias labels loss lse"), (op.backward, "x w bias labels lse dloss dx dw db")):
        names = names.split()
        for bad in names + [None]:
            args = {n: Tensor("float64" if n == bad else types.get(n, "bfloat16"), shapes[n], at=i << 32)
                    for i, n in enumerate(names)}
            with pytest.raises(ops.OperatorError) as e:
                call(**args)
            if bad:
                assert str(e.value).startswith(bad + " is of torch.float64"), (bad, str(e.value))
            else:
                assert "the description says" not in str(e.value), str(e.value)
    with pytest.raises(ops.OperatorError) as e:  # torch's usual labels are of 64 bits
        op.forward(A[0], A[1], Tensor("int64", (M,)), A[2])
    assert "int32" in str(e.value)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_the_workspace_does_for_every_choice_of_gradients(t):
    """A call for some of the gradients takes no more than *_workspace says, which
    is for all of them (another layout of x, other plans)."""
    rng = random.Random(5)
    for _ in range(3000):
        M, K, C = (int(2 ** rng.uniform(0, most)) for most in (8.5, 12, 14))
        odd = rng.choice([0, 0, 3])
        op = ops.CrossEntropy(M, K, C, t, ld_x=K + odd, ld_w=C + rng.choice([0, 3]))
        n = op.workspace_bytes(backward=True)
        for wanted in range(1, 8):
            out = [(1 + i << 52) if wanted >> i & 1 else None for i in range(3)]
            assert op._backward(op._d, *(1 + i << 44 for i in (0, 1)), None, *(3 + i << 44 for i in range(3)), *out, 1 << 58,
                                n, None) == -1
            message = str(op._refused())
            assert "needed are" not in message, (t, M, K, C, odd, wanted, message)
