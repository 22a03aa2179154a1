"""The feed-forward operators (include/volta_ops.h) without a GPU: the header
against the ctypes tables, what calls are refused and with which message, and
the products' plans."""
from __future__ import annotations

import ctypes as C
import os

import numpy as np
import pytest

from tests import ops_ref as R
from tests.test_abi import header_functions
from volta_amd import HIP_LIB, load_hip, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


def test_header_and_ctypes_tables_agree():
    assert sorted(ops.SIGNATURES) == header_functions("volta_ops.h")
    lib = load_hip().lib
    for name in ops.SIGNATURES:
        assert hasattr(lib, name), name


# Addresses that no call may reach: every one is refused on the host.
A = [0x100000000 * (i + 1) for i in range(16)]


def refused(call, *parts):
    with pytest.raises(ops.OperatorError) as e:
        call()
    for p in parts:
        assert p in str(e.value), str(e.value)


def test_descriptions_refused():
    for f, text in [(lambda: ops.Linear(-1, 4, 4), "rows is -1"), (lambda: ops.Linear(4, 0, 4), "inputs is 0"),
                    (lambda: ops.Linear(4, 4, (1 << 21) + 1), "outputs is"), (lambda: ops.Linear(4, 8, 4, ld_x=7), "ld_x is 7"),
                    (lambda: ops.Linear(4, 8, 4, ld_w=(1 << 21) + 1), "ld_w is"),
                    (lambda: ops.GatedFF(4, 4, 0), "hidden is 0"), (lambda: ops.GatedFF(4, 4, 9, ld_pre=8), "ld_pre is 8"),
                    (lambda: ops.RmsNorm(4, 0), "cols is 0"), (lambda: ops.RmsNorm(4, 4, eps=-1.0), "eps"),
                    (lambda: ops.RmsNorm(4, 4, eps=float("nan")), "eps"),
                    (lambda: ops.RmsNorm(4, 4, group=128), "group is 128"),
                    (lambda: ops.RmsNorm(4, 4, out="e4m3", group=64), "group is 64")]:
        op = f()
        refused(op.workspace_bytes, text)
    op = ops.Linear(4, 4, 4)
    op.desc.type = 3
    refused(op.workspace_bytes, "type is 3")
    op.desc.type, op.desc.act = 0, 6
    refused(op.workspace_bytes, "act is 6")
    lib = load_hip().lib
    assert lib.volta_op_linear_workspace(None, 0) == -1 and b"description is NULL" in lib.volta_rt_last_error()
    assert lib.volta_op_linear_workspace(C.byref(ops.Linear(4, 4, 4).desc), 2) == -1
    for p in (-0.1, 1.0, float("nan")):
        refused(lambda: ops.Dropout(4, 4, p=p).forward(A[0], A[1]), "p must be")


def test_pointers_refused():
    lin, gat, nrm, drp = ops.Linear(4, 8, 8), ops.GatedFF(4, 8, 8), ops.RmsNorm(4, 8), ops.Dropout(4, 8)
    refused(lambda: lin.forward(None, A[1], A[2]), "x is NULL")
    refused(lambda: lin.forward(A[0], None, A[2]), "w is NULL")
    refused(lambda: lin.forward(A[0], A[1], None), "y is NULL")
    refused(lambda: lin.forward(A[0] + 2, A[1], A[2]), "x is not aligned")
    refused(lambda: lin.backward(A[0], A[1], A[2], workspace=A[9]), "all NULL")
    refused(lambda: lin.backward(None, A[1], A[2], dx=A[3], workspace=A[9]), "dy is NULL")
    refused(lambda: lin.backward(A[0], None, A[2], dw=A[3], workspace=A[9]), "x is NULL")
    refused(lambda: lin.backward(A[0], A[1], None, dx=A[3], workspace=A[9]), "w is NULL")
    refused(lambda: ops.Linear(4, 8, 8, act="relu").backward(A[0], A[1], A[2], dx=A[3], workspace=A[9]), "pre is NULL")
    refused(lambda: gat.forward(A[0], A[1], A[2], A[3], gate=A[4]), "both or neither")
    refused(lambda: gat.forward(A[0], A[1], None, A[3]), "w_up is NULL")
    refused(lambda: gat.backward(*A[:6], dw_gate=A[6], workspace=A[9]), "both or neither")
    refused(lambda: gat.backward(*A[:6], workspace=A[9]), "every gradient is NULL")
    refused(lambda: gat.backward(*A[:5], None, dx=A[6], workspace=A[9]), "up is NULL")
    refused(lambda: nrm.forward(A[0], None), "y is NULL")
    refused(lambda: nrm.forward(A[0], A[1], scales=A[2]), "E4M3 alone")
    refused(lambda: ops.RmsNorm(4, 8, out="e4m3").forward(A[0], A[1]), "scales is NULL")
    refused(lambda: nrm.backward(A[0], A[1], A[2]), "both NULL")
    refused(lambda: nrm.backward(A[0], A[1], None, dx=A[3]), "rstd is NULL")
    refused(lambda: drp.forward(None, A[1]), "x is NULL")
    for t in ("bf16", "f16"):
        refused(lambda: ops.Dropout(4, 8, t).forward(A[0] + 1, A[1]), "x is not aligned")


def test_workspaces_refused():
    op = ops.Linear(300, 64, 64, act="gelu")
    n = op.workspace_bytes(backward=True)
    assert n >= 300 * 64 * 4
    lib, d = load_hip().lib, C.byref(op.desc)
    args = [d, A[0], A[1], A[2], A[3], A[4], A[5], A[6]]
    for ws, have, text in ((None, n, b"holds 0 bytes"), (A[9], n - 1, b"needed are"), (A[9] + 8, n, b"16-byte")):
        assert lib.volta_op_linear_backward(*args, ws, have, None) == -1
        assert text in lib.volta_rt_last_error()
    nrm = ops.RmsNorm(4, 8)
    refused(lambda: nrm.backward(A[0], A[1], A[2], dweight=A[3]), "workspace holds 0")


def test_overlaps_refused():
    lin = ops.Linear(4, 8, 8)
    refused(lambda: lin.forward(A[0], A[1], A[0]), "x and y overlap")
    refused(lambda: lin.forward(A[0], A[1], A[1] + 32), "w and y overlap")
    refused(lambda: lin.forward(A[0], A[1], A[2], pre=A[2]), "y and pre overlap")
    refused(lambda: lin.forward(A[0], A[1], A[2], residual=A[2] + 4), "residual and y overlap")
    refused(lambda: ops.Linear(4, 8, 8, ld_y=9).forward(A[0], A[1], A[2], residual=A[2]), "residual and y overlap")
    refused(lambda: ops.Linear(4, 8, 8, act="relu").backward(*A[:4], dx=A[4], dw=A[5], workspace=A[5] - 64),
            "overlaps the workspace")
    refused(lambda: lin.backward(*A[:3], dx=A[4], dw=A[4] + 64, workspace=A[9]), "dx and dw overlap")
    refused(lambda: ops.RmsNorm(4, 8).forward(A[0], A[0]), "x and y overlap")
    refused(lambda: ops.RmsNorm(4, 8, ld_sum=16).forward(A[0], A[1], sum=A[0]), "x and sum overlap")
    refused(lambda: ops.Dropout(4, 8).forward(A[0], A[0] + 4), "x and y overlap")
    # halves of one wider matrix lie beside each other, shifted ones do not
    wide = ops.GatedFF(4, 8, 8, ld_w=16, ld_pre=16, ld_dw=16)
    refused(lambda: wide.forward(A[0], A[1], A[1] + 32, A[2], gate=A[3], up=A[3] + 28), "gate and up overlap")
    refused(lambda: wide.forward(A[0], A[1], A[1] + 32, A[2], gate=A[3], up=A[3] + 36), "gate and up overlap")


def plan(e, layout, kind, M, N, K, pieces=1, outputs=1, direct=1):
    out = (C.c_int32 * 3)()
    load_hip().lib.volta_hip_op_plan(e, layout, kind, M, N, K, pieces, outputs, direct, out)
    return list(out)


def test_plans_cover_the_sum():
    """Over a grid of sizes: the splits' stages cover the sum without an empty
    split, a plan fits its kernel (tiles 0, 1 and 3 load directly, the skinny ones
    from 5 on are not for dW), and the partial sums stay under a GiB."""
    rng = np.random.default_rng(0)
    for _ in range(3000):
        e, direct = int(rng.choice([2, 4])), int(rng.integers(2))
        layout = int(rng.integers(3))
        kind = 2 if layout else int(rng.integers(2))
        M, N, K = (int(2 ** rng.uniform(0, 15)) for _ in range(3))
        pieces, outputs = (2 if layout == 1 and rng.random() < 0.5 else 1), (2 if layout == 2 and rng.random() < 0.5 else 1)
        tile, splits, per = plan(e, layout, kind, M, N, K, pieces, outputs, direct)
        stages = pieces * -(-K // (128 // e))
        assert splits >= 1 and (splits - 1) * per < stages <= splits * per, (M, N, K, splits, per)
        assert tile not in (0, 1, 3) or direct
        assert tile < 5 or layout != 2
        if splits > 1:
            assert 4 * splits * (2 if kind == 1 else outputs) * M * N < 1 << 30


def test_workspace_holds_either_form():
    """The workspace does not depend on the pointers' alignment, which is not known yet."""
    for M, K, N in ((1, 4096, 512), (100, 4096, 96), (2000, 1500, 300)):
        need = 0
        for direct in (0, 1):
            _, splits, _ = plan(2, 0, 0, M, N, K, direct=direct)
            need = max(need, 4 * splits * M * N if splits > 1 else 0)
        assert ops.Linear(M, K, N, "bf16").workspace_bytes() >= need


def test_host_types():
    """The tests' own conversions: to the nearest, ties to even."""
    assert list(R.unpack(R.pack([1 + 2.0**-8, 1 + 3 * 2.0**-8], "bf16"), "bf16")) == [1.0, 1 + 4 * 2.0**-8]
    codes = np.arange(256, dtype=np.uint8)
    v = R.unpack(codes, "e4m3")
    assert v[0x7E] == 448 and v[1] == 2.0**-9 and v[0x88] == -(2.0**-6) and np.isnan(v[0x7F]) and np.isnan(v[0xFF])
    assert list(R.splitmix_keep(4, 0, 0, 0.5)) == [bool(b >= 1 << 31) for z in (0xE220A8397B1DCDAF, 0x6E789E6AA1B965F4)
                                                   for b in (z & 0xFFFFFFFF, z >> 32)]


def test_products_of_too_many_blocks_refused():
    """Whatever the direction: by the workspace's call already."""
    for op in (ops.Linear(1 << 30, 64, 64, "bf16"), ops.GatedFF(1 << 30, 64, 64, "bf16"),
               ops.Linear(1 << 30, 63, 65, "f32", act="gelu")):
        for backward in (False, True):
            refused(lambda: op.workspace_bytes(backward=backward), "too many")
    assert ops.Linear(1 << 24, 64, 64, "bf16").workspace_bytes(backward=True) > 0
