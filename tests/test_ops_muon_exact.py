"""Muon's choice of exact bfloat16 updates (include/volta_ops.h) without a GPU."""
from __future__ import annotations

import os

import pytest

from tests.test_ops import refused
from volta_amd import HIP_LIB, ops

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libvolta_hip.so not built")


@pytest.mark.parametrize("m,n", [(64, 64), (300, 301), (512, 2000), (4096, 1024)])
def test_exact_bfloat16_is_held_as_the_other_types_are(m, n):
    def space(t, **kw):
        return ops.Muon(m, n, t, **kw).workspace_bytes()

    assert space("bf16", exact=True) == space("f16") == space("f16", exact=True) == space("f32")
    if min(m, n) > 96:  # smaller ones always are
        assert space("bf16") < space("bf16", exact=True)
    else:
        assert space("bf16") == space("bf16", exact=True)


def test_other_values_refused():
    op = ops.Muon(4, 4, "bf16")
    op.desc.exact = 2
    refused(op.workspace_bytes, "exact is 2")
