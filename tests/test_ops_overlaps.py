"""Which matrices of a call of the operators may be one: the two that the call
names, not a third at the same address.  Without a GPU."""
from __future__ import annotations

import os

import pytest

from tests.test_ops import A, refused
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def test_a_third_matrix_at_the_same_address_is_refused():
    lin = ops.Linear(4, 8, 8)
    refused(lambda: lin.forward(A[0], A[1], A[0], residual=A[0]), "x and y overlap")
    refused(lambda: ops.Linear(1, 8, 8).forward(A[0], A[1], A[2], bias=A[2], residual=A[2]), "bias and y overlap")
    refused(lambda: ops.RmsNorm(4, 8).backward(A[0], A[1], A[2], dx=A[0], dsum=A[0]), "dy and dx overlap")
    refused(lambda: ops.RmsNorm(1, 8).forward(A[0], A[1], weight=A[0], sum=A[0]), "weight and sum overlap")
    refused(lambda: ops.Linear8(1, 16, 8).forward(A[0], A[1], A[2], A[3], A[4], bias=A[4], residual=A[4], workspace=A[9]),
            "bias and y overlap")


def test_the_named_ones_are_taken():
    for call in (lambda: ops.Linear(4, 8, 8).forward(A[0], A[1], A[2], residual=A[2]),
                 lambda: ops.RmsNorm(4, 8).forward(A[0], A[1], residual=A[0], sum=A[0]),
                 lambda: ops.RmsNorm(4, 8).backward(A[0], A[1], A[2], dx=A[3], dsum=A[3]),
                 lambda: ops.Dropout(4, 8).forward(A[0], A[0], residual=A[0])):
        with pytest.raises(ops.OperatorError) as e:
            call()
        assert "overlap" not in str(e.value)
