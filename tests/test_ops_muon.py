"""The update by orthogonalised momentum (include/volta_ops.h) without a GPU:
what is refused, with which message."""
from __future__ import annotations

import os

import pytest

from tests.test_ops import A, refused
from tests.test_ops_matrices import Tensor
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def test_descriptions_refused():
    for f, text in [(lambda: ops.Muon(0, 4), "rows is 0"), (lambda: ops.Muon(4, 0), "cols is 0"),
                    (lambda: ops.Muon(4, 4, batch=0), "batch is 0"), (lambda: ops.Muon(4, 4, batch=65536), "batch is"),
                    (lambda: ops.Muon(1 << 21, 4, batch=1024), "batch times rows"),
                    (lambda: ops.Muon(4, 4, steps=0), "steps is 0"), (lambda: ops.Muon(4, 4, steps=65), "steps is 65"),
                    (lambda: ops.Muon(4, 8, ld_u=7), "ld_u is 7"), (lambda: ops.Muon(4, 8, ld_m=7), "ld_m is 7"),
                    (lambda: ops.Muon(4, 8, ld_o=7), "ld_o is 7"), (lambda: ops.Muon(4, 4, eps=-1.0), "eps"),
                    (lambda: ops.Muon(4, 4, eps=float("nan")), "eps"),
                    (lambda: ops.Muon(4, 4, coefficients=(1.0, float("inf"), 0.0)), "coefficient"),
                    (lambda: ops.Muon(4, 4, "bf16", coefficients=(3.0, 1.0, 1.0)), "past 1024"),
                    (lambda: ops.Muon(4, 4, "f32", coefficients=(3.0, 1.0, 1.0)), "past 1024"),
                    (lambda: ops.Muon(1 << 21, 1 << 21, "bf16"), "too many")]:
        refused(lambda: f().workspace_bytes(), text)
    op = ops.Muon(4, 4)
    op.desc.type = 3
    refused(op.workspace_bytes, "type is 3")


def test_calls_refused():
    op = ops.Muon(4, 8, "bf16")
    refused(lambda: op.orthogonalize(None, A[1], workspace=A[9]), "u is NULL")
    refused(lambda: op.orthogonalize(A[0], None, workspace=A[9]), "o is NULL")
    refused(lambda: op.orthogonalize(A[0], A[0] + 2, workspace=A[9]), "u and o overlap")
    refused(lambda: ops.Muon(4, 8, "bf16", ld_o=9).orthogonalize(A[0], A[0], workspace=A[9]), "u and o overlap")
    refused(lambda: op.orthogonalize(A[0], A[1]), "workspace holds 0")
    refused(lambda: op.orthogonalize(A[0], A[1], workspace=A[1]), "overlaps the workspace")
    for i, name in enumerate(("w", "g", "m")):
        args = [A[0], A[1], A[2]]
        args[i] = None
        refused(lambda: op.step(*args, 0.1, workspace=A[9]), name + " is NULL")
    refused(lambda: op.step(A[0], A[1], A[2] + 2, 0.1, workspace=A[9]), "m is not aligned")
    refused(lambda: op.step(A[0], A[0], A[2], 0.1, workspace=A[9]), "g and w_out overlap")
    f32 = ops.Muon(4, 8)
    refused(lambda: f32.step(A[0], A[1], A[1], 0.1, workspace=A[9]), "g and m_out overlap")
    refused(lambda: f32.step(A[0], A[1], A[0], 0.1, workspace=A[9]), "overlap")
    refused(lambda: op.step(A[0], A[1], A[2], 0.1, w_out=A[0] + 2, workspace=A[9]), "w and w_out overlap")
    refused(lambda: op.step(A[0], A[1], A[2], 0.1, momentum_out=A[1], workspace=A[9]), "g and m_out overlap")
    refused(lambda: op.step(A[0], A[1], A[2], float("nan"), workspace=A[9]), "not finite")
    refused(lambda: op.step(A[0], A[1], A[2], 0.1, beta=float("inf"), workspace=A[9]), "not finite")


def test_every_matrix_is_compared():
    op = ops.Muon(6, 10, "bf16", batch=3)
    f32 = ("momentum", "momentum_out")
    for call, names, extra in ((op.orthogonalize, ("u", "o"), {}), (op.step, ("w", "g", "momentum", "w_out", "momentum_out"),
                                                                    {"lr": 0.1})):
        for bad in names + (None,):
            args = {n: Tensor("float64" if n == bad else "float32" if n in f32 else "bfloat16", (3, 6, 10), at=i << 32)
                    for i, n in enumerate(names)}
            with pytest.raises(ops.OperatorError) as e:
                call(**args, **extra)
            if bad:
                assert str(e.value).startswith(bad + " is of torch.float64"), (bad, str(e.value))
            else:
                assert "the description says" not in str(e.value), str(e.value)
    with pytest.raises(ops.OperatorError):  # a matrix of the batch is missing
        op.orthogonalize(Tensor("bfloat16", (2, 6, 10)), A[1])


def test_both_forms_are_planned():
    """Two steps at once take three matrices of the smaller side, one by one two:
    wide and tall matrices the first, square ones the second."""
    for batch, m, n, pairs in ((16, 512, 2000, True), (1, 4096, 16384, True), (1, 16384, 4096, True), (1, 512, 2000, False),
                               (1, 1024, 1024, False), (1, 301, 300, False)):
        (m8, n8), lines = [-(-v // 8) * 8 for v in (m, n)], lambda v: -(-v // 64) * 64  # whole chunks, whole cache lines
        small = ops.Muon(m, n, "bf16", batch=batch).workspace_bytes() // batch - 2 * 2 * m8 * lines(n8)
        assert (small >= 3 * 2 * min(m8, n8) * lines(min(m8, n8))) == pairs, (batch, m, n, small)
    # a single step has nothing to go with
    one, two = (ops.Muon(512, 2000, "bf16", batch=16, steps=s).workspace_bytes() for s in (1, 2))
    assert one < two
