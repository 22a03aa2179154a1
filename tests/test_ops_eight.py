"""e4m3 codes and the linear layer of them (include/volta_ops.h) without a GPU:
what is refused, with which message, and what is planned."""
from __future__ import annotations

import os

import pytest

from tests.test_ops import A, plan, refused
from tests.test_ops_matrices import Tensor
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def test_descriptions_refused():
    for f, text in [(lambda: ops.Linear8(-1, 4, 4), "rows is -1"), (lambda: ops.Linear8(4, 0, 4), "inputs is 0"),
                    (lambda: ops.Linear8(4, 4, 0), "outputs is 0"), (lambda: ops.Linear8(4, 8, 4, ld_x=7), "ld_x is 7"),
                    (lambda: ops.Linear8(4, 8, 4, ld_w=7), "ld_w is 7"), (lambda: ops.Linear8(4, 8, 4, ld_y=3), "ld_y is 3"),
                    (lambda: ops.Linear8(4, 8, 4, ld_residual=3), "ld_residual is 3"),
                    (lambda: ops.Linear8(4, 8, 4, group=64), "group is 64"),
                    (lambda: ops.Linear8(1 << 30, 64, 64), "too many")]:
        refused(lambda: f().workspace_bytes(), text)
    for f, text in [(lambda: ops.Quantize(-1, 4), "rows is -1"), (lambda: ops.Quantize(4, 0), "cols is 0"),
                    (lambda: ops.Quantize(4, 8, ld_x=7), "ld_x is 7"), (lambda: ops.Quantize(4, 8, ld_y=7), "ld_y is 7"),
                    (lambda: ops.Quantize(8, 4, by="blocks", ld_y=7), "ld_y is 7"),
                    (lambda: ops.Quantize((1 << 21) + 1, 4, by="blocks"), "rows is")]:
        refused(lambda: f().forward(A[0], A[1], A[2]), text)
    q = ops.Quantize(4, 8)
    q.desc.groups = 2
    refused(lambda: q.forward(A[0], A[1], A[2]), "groups is 2")
    q.desc.groups, q.desc.type = 0, 3
    refused(lambda: q.forward(A[0], A[1], A[2]), "type is 3")
    op = ops.Linear8(4, 8, 8)
    op.desc.type = 3
    refused(op.workspace_bytes, "type is 3")
    op.desc.type, op.desc.act = 1, 6
    refused(op.workspace_bytes, "act is 6")


def test_calls_refused():
    q, b = ops.Quantize(4, 8), ops.Quantize(4, 8, by="blocks")
    for op in (q, b):
        refused(lambda: op.forward(None, A[1], A[2]), "x is NULL")
        refused(lambda: op.forward(A[0], None, A[2]), "y is NULL")
        refused(lambda: op.forward(A[0], A[1], None), "scales is NULL")
        refused(lambda: op.forward(A[0] + 2, A[1], A[2]), "x is not aligned")
        refused(lambda: op.forward(A[0], A[0] + 8, A[2]), "x and y overlap")
        refused(lambda: op.forward(A[0], A[1], A[1] + 8), "y and scales overlap")
    op = ops.Linear8(4, 16, 8, "f32")
    args = [A[0], A[1], A[2], A[3], A[4]]
    for i, name in enumerate(("x", "x_scales", "w", "w_scales", "y")):
        some = list(args)
        some[i] = None
        refused(lambda: op.forward(*some, workspace=A[9]), name + " is NULL")
    refused(lambda: op.forward(A[0], A[1] + 2, *args[2:], workspace=A[9]), "x_scales is not aligned")
    refused(lambda: op.forward(*args[:4], A[2], workspace=A[9]), "w and y overlap")
    refused(lambda: op.forward(*args, residual=A[4] + 4, workspace=A[9]), "residual and y overlap")
    odd = ops.Linear8(2000, 8200, 4096, "f16")
    assert odd.workspace_bytes() >= (2000 + 4096) * 8208  # both laid out anew
    refused(lambda: odd.forward(*args), "workspace holds 0")


def test_plans_cover_the_sum():
    for M in (1, 16, 100, 300, 2048, 8192):
        for K in (1, 128, 1000, 16384):
            for N in (8, 1000, 4096, 16384):
                for direct in (0, 1):
                    tile, splits, per = plan(1, 1, 0, M, N, K, direct=direct)
                    stages = -(-K // 128)
                    assert (splits - 1) * per < stages <= splits * per
                    assert tile not in (0, 1, 3) or direct


def test_every_matrix_is_compared():
    M, K, N = 4, 200, 300
    shapes = {"x": (M, K), "x_scales": (M, 2), "w": (N, K), "w_scales": (3, 2), "y": (M, N), "bias": (N,),
              "residual": (M, N)}
    types = {"x": "float8_e4m3fn", "w": "uint8", "x_scales": "float32", "w_scales": "float32"}
    q, b = {"x": (M, K), "y": (M, K), "scales": (M, 2)}, {"x": (M, K), "y": (K, M), "scales": (2, 1)}
    codes = {"y": "float8_e4m3fn", "scales": "float32"}
    for call, shape, type in ((ops.Linear8(M, K, N, "bf16").forward, shapes, types),
                              (ops.Quantize(M, K, "bf16").forward, q, codes),
                              (ops.Quantize(M, K, "bf16", by="blocks").forward, b, codes)):
        for bad in list(shape) + [None]:
            args = {n: Tensor("float64" if n == bad else type.get(n, "bfloat16"), shape[n], at=i << 32)
                    for i, n in enumerate(shape)}
            with pytest.raises(ops.OperatorError) as e:
                call(**args)
            if bad:
                assert str(e.value).startswith(bad + " is of torch.float64"), (bad, str(e.value))
            else:
                assert "the description says" not in str(e.value), str(e.value)
