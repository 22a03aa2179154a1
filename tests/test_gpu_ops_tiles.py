"""The kernels of the operators' products (volta_amd/csrc/ops_gemm.h), tile by
tile: which plans they take."""
from __future__ import annotations

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import Mat
from tests.test_gpu_ops import GATED, LINEAR, NN, NT, STORE, TILES, TN, whole
from volta_amd import load_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return load_hip()


@pytest.mark.parametrize("t", R.TYPES)
def test_tiles_without_a_staged_form_refused(lib, t):
    """256x256, 256x128 and 64x128 take direct loads alone, and dW no tile of
    few rows: another tile in their place would go unnoticed."""
    M, K, N = 40, 64, 48
    rng = np.random.default_rng(1)
    forms = ((NN, LINEAR), (NN, GATED), (NT, STORE), (TN, STORE))
    for layout, kind in forms:
        P = Mat(lib, t, *((K, M) if layout == TN else (M, K)), whole(rng, *((K, M) if layout == TN else (M, K))))
        Q = Mat(lib, t, *((N, K) if layout == NT else (K, N)), whole(rng, *((N, K) if layout == NT else (K, N))))
        for tile in TILES:
            out = Mat(lib, t, M, N)
            few = tile.startswith("skinny") and layout == TN
            for direct in (0, 1):
                rc = lib.lib.volta_hip_op_product(R.TYPES.index(t), layout, kind, TILES[tile], 1, direct, P.ptr, P.ptr,
                                                  P.ld, Q.ptr, Q.ptr, Q.ld, out.ptr, out.ptr, out.ld, M, N, K, 1, 1)
                taken = not few and (direct or tile not in ("256", "256x128", "64x128"))
                assert (rc == 0) == bool(taken), (layout, kind, tile, direct)
                assert taken or out.untouched(), (layout, kind, tile, direct)
