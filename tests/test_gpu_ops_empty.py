"""Calls of no rows whose row-shaped matrices are NULL, as empty tensors are, on the
GPU: they return, and weights' gradients are zero."""
from __future__ import annotations

import numpy as np
import pytest

from tests.ops_ref import TYPES, Mat
from tests.test_gpu_ops import Space
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
def test_no_rows(t):
    lib = load_hip()
    K, C = 24, 40
    w, wide = Mat(lib, t, K, C, np.ones((K, C))), Mat(lib, t, 1, C, np.ones(C))
    dw, db = Mat(lib, t, K, C), Mat(lib, t, 1, C)
    op = ops.CrossEntropy(0, K, C, t)
    op.forward(None, w, None, None, workspace=Space(lib, op))
    ws = Space(lib, op, True)
    op.backward(None, w, None, None, None, workspace=ws)
    op.backward(None, w, None, None, None, dw=dw, db=db, workspace=ws)
    assert not dw.get().any() and not db.get().any()
    op = ops.Linear(0, K, C, t, "gelu")
    ws = Space(lib, op, True)
    op.forward(None, w, None, workspace=Space(lib, op))
    op.backward(None, None, w, workspace=ws)
    dw, db = Mat(lib, t, K, C), Mat(lib, t, 1, C)
    op.backward(None, None, w, dw=dw, db=db, workspace=ws)
    assert not dw.get().any() and not db.get().any()
    op = ops.GatedFF(0, K, C, t)
    op.forward(None, w, w, None, workspace=Space(lib, op))
    op.backward(None, None, w, w, None, None, workspace=Space(lib, op, True))
    op, dweight = ops.RmsNorm(0, C, t), Mat(lib, t, 1, C)
    op.forward(None, None, weight=wide)
    ws = Space(lib, op, True)
    op.backward(None, None, None, weight=wide, workspace=ws)
    op.backward(None, None, None, weight=wide, dweight=dweight, workspace=ws)
    assert not dweight.get().any()
    ops.Quantize(0, K, t).forward(None, None, None)
    ops.Quantize(0, K, t, by="blocks").forward(None, None, None)
