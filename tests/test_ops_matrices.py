"""What volta_amd.ops compares of the matrices it is handed with an operator's
description, before the library sees an address: without a GPU."""
from __future__ import annotations

import os

import pytest

from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")

ADDRESS = 0x7F0000000000


class Tensor:
    """What the operators read of a torch tensor."""

    def __init__(self, dtype, shape, strides=None, at=0):
        self.dtype, self.shape, self.at = "torch." + dtype, tuple(shape), ADDRESS + at
        packed = [1]
        for n in reversed(self.shape[1:]):
            packed.insert(0, packed[0] * n)
        self.packed = tuple(packed[:len(self.shape)])
        self.strides = tuple(strides) if strides is not None else self.packed

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return self.strides == self.packed

    @property
    def nbytes(self):
        n = {"torch.float64": 8, "torch.float32": 4, "torch.uint8": 1}.get(self.dtype, 2)
        for d in self.shape:
            n *= d
        return n

    def data_ptr(self):
        return self.at


class Array:
    """What they read of a DeviceArray."""

    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, ADDRESS


def read(m, type="bf16", rows=4, cols=8, ld=0):
    return ops._matrix("x", ops.TYPES[type], rows, cols, ld)(m)


def refused(m, text, **kw):
    with pytest.raises(ops.OperatorError) as e:
        read(m, **kw)
    assert "x " in str(e.value) and text in str(e.value), str(e.value)


@pytest.mark.parametrize("m", [Tensor("bfloat16", (4, 8)), Tensor("bfloat16", (2, 2, 8)), Tensor("bfloat16", (9, 8)),
                               Tensor("bfloat16", (32,)), Tensor("bfloat16", (1, 4, 1, 8)), Array(64), Array(100)])
def test_packed_matrices_taken(m):
    assert read(m) == ADDRESS
    assert read(m) == ADDRESS


def test_rows_apart_taken():
    for m in (Tensor("bfloat16", (4, 8), (16, 1)), Tensor("bfloat16", (2, 2, 8), (32, 16, 1)),
              Tensor("bfloat16", (56,)), Tensor("bfloat16", (1, 5, 8), (7, 16, 1)), Array(2 * 56)):
        assert read(m, ld=16) == ADDRESS
    assert read(Tensor("float32", (300, 1), (7, 1)), type="f32", rows=300, cols=1, ld=7) == ADDRESS
    assert read(Tensor("float32", (300,), (7,)), type="f32", rows=300, cols=1, ld=7) == ADDRESS
    # one row: how far the next one would be has no say
    assert read(Tensor("float16", (2, 8), (24, 1)), type="f16", rows=1, ld=16) == ADDRESS


def test_a_row_by_its_bytes():
    """Of one row, and of a vector, any packed tensor of as many elements."""
    for rows_of_one in (ops._matrix("x", ops.TYPES["bf16"], 1, 8), ops._matrix("x", ops.TYPES["bf16"], 1, 8, 8)):
        for m in (Tensor("bfloat16", (8,)), Tensor("bfloat16", (1, 8)), Tensor("bfloat16", (1, 1, 8)), Tensor("bfloat16", (9,))):
            assert rows_of_one(m) == ADDRESS and rows_of_one(m) == ADDRESS
        for m in (Tensor("bfloat16", (7,)), Tensor("bfloat16", (8,), (2,)), Tensor("float32", (4,)), Tensor("float16", (8,)),
                  Tensor("bfloat16", (2, 4), (8, 1))):
            with pytest.raises(ops.OperatorError):
                rows_of_one(m)


def test_raw_addresses_none_and_no_rows_taken():
    assert read(ADDRESS) == ADDRESS and read(None) is None
    assert read(Tensor("bfloat16", (0, 8)), rows=0) == ADDRESS and read(Array(4), rows=0) == ADDRESS
    assert read(Tensor("uint8", (4, 8)), type="e4m3") == read(Tensor("float8_e4m3fn", (4, 8)), type="e4m3") == ADDRESS


def test_other_types_refused():
    for type, names in (("f32", ("bfloat16", "float64")), ("bf16", ("float16", "float32")), ("f16", ("bfloat16", "int16")),
                        ("e4m3", ("float8_e5m2", "bfloat16", "float8_e4m3fnuz"))):
        for n in names:
            refused(Tensor(n, (4, 8)), "the description says " + type, type=type)
    # and after one that was taken
    x = ops._matrix("x", ops.TYPES["bf16"], 4, 8)
    assert x(Tensor("bfloat16", (4, 8))) == ADDRESS
    with pytest.raises(ops.OperatorError):
        x(Tensor("float32", (4, 8)))


@pytest.mark.parametrize("m", [Tensor("bfloat16", (8, 4), (1, 8)), Tensor("bfloat16", (8, 4)), Tensor("bfloat16", (3, 8)),
                               Tensor("bfloat16", (31,)), Tensor("bfloat16", (4, 8), (16, 1)), Tensor("bfloat16", (4, 8), (0, 1)),
                               Tensor("bfloat16", (4, 8), (16, 2)), Tensor("bfloat16", (2, 2, 8), (64, 8, 1)),
                               Tensor("bfloat16", (64,), (2,)), Tensor("bfloat16", (0,)), Tensor("bfloat16", (0, 8)),
                               Tensor("bfloat16", ())])
def test_transposed_strided_and_short_tensors_refused(m):
    refused(m, "4 rows of 8, 8 apart")


def test_other_distances_refused():
    for m in (Tensor("bfloat16", (4, 8)), Tensor("bfloat16", (4, 8), (24, 1)), Tensor("bfloat16", (55,)),
              Tensor("bfloat16", (2, 2, 8), (16, 16, 1))):
        refused(m, "16 apart", ld=16)


def test_short_arrays_refused():
    refused(Array(63), "holds 63 bytes, the description says 64")
    refused(Array(111), "says 112", ld=16)


def test_every_matrix_of_every_call_is_compared():
    """Each argument in turn of the wrong type: the message names it, whatever
    the others are."""
    M, K, N = 4, 16, 24
    lin, gat, drp = ops.Linear(M, K, N, "bf16"), ops.GatedFF(M, K, N, "bf16"), ops.Dropout(M, N, "bf16")
    nrm, codes = ops.RmsNorm(M, N, "bf16"), ops.RmsNorm(M, 300, "bf16", out="e4m3", group=128)
    wide = {"x": (M, 300), "y": (M, 300), "residual": (M, 300), "sum": (M, 300), "weight": (300,), "rstd": (M,),
            "scales": (M, 3)}
    row, vec = {"x": (M, K), "dx": (M, K)}, (N,)
    shapes = {**row, **dict.fromkeys(("w", "dw", "w_gate", "w_up", "dw_gate", "dw_up"), (K, N)),
              **dict.fromkeys(("bias", "db", "b_gate", "b_up", "db_gate", "db_up"), vec),
              **dict.fromkeys(("y", "dy", "residual", "pre", "h", "dh", "gate", "up"), (M, N))}
    normed = {**dict.fromkeys(("dy", "s", "dsum", "dx"), (M, N)), "rstd": (M,), "weight": vec, "dweight": vec}
    dropped = dict.fromkeys(("x", "y", "residual", "dy", "dx"), (M, N))
    for call, names, shape in (
            (lin.forward, "x w y bias residual pre", shapes), (lin.backward, "dy x w pre dx dw db", shapes),
            (gat.forward, "x w_gate w_up h b_gate b_up gate up", shapes),
            (gat.backward, "dh x w_gate w_up gate up dx dw_gate dw_up db_gate db_up", shapes),
            (codes.forward, "x y weight residual sum rstd scales", wide),
            (nrm.backward, "dy s rstd dx weight dsum dweight", normed), (drp.forward, "x y residual", dropped),
            (drp.backward, "dy dx", dropped)):
        names = names.split()
        for bad in names + [None]:
            args = {}
            for i, n in enumerate(names):
                t = "float32" if n in ("rstd", "scales") else "uint8" if call == codes.forward and n == "y" else "bfloat16"
                args[n] = Tensor("float64" if n == bad else t, shape[n], at=i << 32)
            with pytest.raises(ops.OperatorError) as e:
                call(**args)
            if bad:
                assert str(e.value).startswith(bad + " is of torch.float64"), (bad, str(e.value))
            else:  # all of them right: it is the library that refuses them
                assert "the description says" not in str(e.value), str(e.value)


def test_torch_tensors():
    """Of torch's own: views of a wider matrix, a transposed weight, a slice of
    a prompt, a tensor of another type."""
    torch = pytest.importorskip("torch")
    op = ops.Linear(6, 16, 24, "bf16", ld_w=48)
    w, x, y = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((16, 48), (2, 3, 16), (6, 24)))

    def said(**kw):
        args = {"x": x, "w": w[:, 24:], "y": y, **kw}
        with pytest.raises(ops.OperatorError) as e:
            op.forward(**args)
        return str(e.value)

    assert "the description says" not in said()  # host memory: the library's own check
    assert said(w=w).startswith("w has shape (16, 48)")
    assert said(w=w[:, :24].contiguous()).startswith("w has shape")
    assert said(x=x.float()).startswith("x is of torch.float32")
    assert said(x=x[:, 1:]).startswith("x has shape (2, 2, 16)")
    assert said(y=torch.zeros(24, 6, dtype=torch.bfloat16).t()).startswith("y has shape (6, 24) and strides (1, 6)")
