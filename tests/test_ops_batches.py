"""A batch's matrices as a tensor of three dimensions (volta_amd.ops): compared in
as few steps as one of two."""
from __future__ import annotations

import pytest

from tests.test_ops_matrices import Tensor
from volta_amd import ops


class Counting(Tensor):
    """A tensor that counts how often its strides are asked for."""

    asked = 0

    def stride(self):
        self.asked += 1
        return self.strides


def test_packed_batches_are_compared_without_strides():
    take = ops._matrix("u", ops.TYPES["bf16"], 12, 8)
    seen = Counting("bfloat16", (3, 4, 8))
    dtype = seen.dtype
    for shape, asks in (((3, 4, 8), 1), ((3, 4, 8), 0), ((12, 8), 0), ((2, 6, 8), 0), ((2, 3, 2, 8), 0),
                        ((96,), 1), ((4, 4, 8), 1)):
        m = Counting("bfloat16", shape)
        m.dtype = dtype
        assert take(m) == m.at and m.asked == asks, (shape, m.asked)
    for shape, strides in (((3, 4, 4), None), ((3, 2, 8), None), ((3, 4, 8), (64, 8, 1)), ((6, 2, 4, 2), None)):
        m = Counting("bfloat16", shape, strides)
        m.dtype = dtype
        with pytest.raises(ops.OperatorError, match="u has shape"):
            take(m)


def test_rows_apart_are_compared_by_their_strides():
    take = ops._matrix("u", ops.TYPES["bf16"], 12, 8, 16)
    for _ in range(2):
        m = Counting("bfloat16", (3, 4, 8), (64, 16, 1))
        assert take(m) == m.at
        with pytest.raises(ops.OperatorError):
            take(Counting("bfloat16", (3, 4, 8)))
