"""The update by orthogonalised momentum (volta_amd.ops.Muon) of matrices of few
directions and of far apart ones, whose small directions the steps enlarge most,
on the GPU, held in two numbers and, in larger bfloat16 that is not to be exact, in one.

Tolerances: limits in percent of the norm, whatever the kernels round.  Of two
numbers 0.02 % before the result's rounding (what sums in 32 bits leave of matrices
of rank 1, whose noise is enlarged 484 times: a step's float32 products on the CPU
leave up to 0.015 %).  Of one number what the description's table says, and a
quarter more.  The rounding: of a value in [2^e, 2^(e+1)) evenly over a step, so
step^2 / 12 of its square at most, 2 HALF / sqrt(12) of the norm; a tenth more for
chance, over 4000 values or more."""
from __future__ import annotations

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import HALF, TYPES, Mat
from tests.test_gpu_ops import Layout, say
from tests.test_gpu_ops_muon import iterate, space
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
TWO = 2e-4
# of one number, by the start of a matrix' name
ONE = {"noise": 0.18, "rank 1": 10, "rank 4": 7, "rank r": 5.2, "third": 3, "1 / i^1": 0.4, "1 / i^2": 2, "1 / i^4": 4.6,
       "noise and 4 at 5": 0.4, "noise and 4 at 50": 2.5, "noise and 4 at 500": 7}


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def limit(t, want, before=TWO):
    return (before + 1.1 * 2 * HALF[t] / np.sqrt(12)) * np.linalg.norm(want) + R.FLOOR[t] * np.sqrt(want.size)


def spectra(rng, m, n):
    """Matrices of some directions, of falling ones, of noise beside strong ones."""
    small = min(m, n)
    yield "noise", rng.standard_normal((m, n))
    for name, r in (("rank 1", 1), ("rank 4", 4), ("rank r", max(5, small // 16)), ("third", small // 3)):
        yield name, rng.standard_normal((m, r)) @ rng.standard_normal((r, n))
    u, _, v = np.linalg.svd(rng.standard_normal((m, n)), full_matrices=False)
    for power in (1, 2, 4):
        yield "1 / i^%d" % power, (u * np.arange(1.0, small + 1) ** -power) @ v
    for weight in (5, 50, 500):
        yield "noise and 4 at %d" % weight, (rng.standard_normal((m, n))
                                             + weight * rng.standard_normal((m, 4)) @ rng.standard_normal((4, n)))


SIZES = [(64, 64), (80, 1000), (104, 128), (300, 301), (512, 1024), (1000, 136), (97, 2000), (1024, 640)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("t", TYPES)
def test_orthogonalize(lib, t, m, n):
    op, one = ops.Muon(m, n, t, exact=True), ops.Muon(m, n, t)
    ws, o = space(lib, op), Mat(lib, t, m, n)
    assert (t == "bf16" and min(m, n) > 96) or one.workspace_bytes() == op.workspace_bytes()
    for name, v in spectra(np.random.default_rng(m + n), m, n):
        say(t, m, n, name)
        v = R.unpack(R.pack(v, t), t)
        u, want = Mat(lib, t, m, n, v), iterate(v)
        op.orthogonalize(u, o, workspace=ws)
        assert np.linalg.norm(o.get() - want) <= limit(t, want), name
        before = o.bits()
        one.orthogonalize(u, o, workspace=ws)
        if t == "bf16" and min(m, n) > 96:
            assert np.linalg.norm(o.get() - want) <= limit(t, want, 1.25 * ONE[name] / 100), name
        else:
            assert np.array_equal(o.bits(), before), name
    ws.check()


@pytest.mark.parametrize("steps", [1, 2, 3, 4])
@pytest.mark.parametrize("m,n", [(40, 70), (128, 136), (600, 200)])
@pytest.mark.parametrize("t", TYPES)
def test_any_number_of_steps(lib, t, m, n, steps):
    """One step alone, pairs of them, and both; of a batch whose matrices differ."""
    rng = np.random.default_rng(steps)
    v = np.stack([rng.standard_normal((m, r)) @ rng.standard_normal((r, n)) for r in (1, 8, 30)])
    v = R.unpack(R.pack(v, t), t)
    op = ops.Muon(m, n, t, batch=3, steps=steps, exact=True)
    o = Mat(lib, t, 3 * m, n)
    op.orthogonalize(Mat(lib, t, 3 * m, n, v.reshape(-1, n)), o, workspace=space(lib, op))
    for got, u in zip(o.get().reshape(v.shape), v):
        want = iterate(u, steps=steps)
        assert np.linalg.norm(got - want) <= limit(t, want)


@pytest.mark.parametrize("t", TYPES)
def test_step(lib, t):
    """The weights' update of a gradient of 16 directions."""
    m, n = 512, 768
    rng = np.random.default_rng(4)
    g = R.unpack(R.pack(rng.standard_normal((m, 16)) @ rng.standard_normal((16, n)), t), t)
    zeros, w, mom = np.zeros((m, n)), Mat(lib, t, m, n), Mat(lib, "f32", m, n)
    op = ops.Muon(m, n, t, exact=True)
    op.step(Mat(lib, t, m, n, zeros), Mat(lib, t, m, n, g), Mat(lib, "f32", m, n, zeros), 0.5, beta=0.5, scale=2.0,
            w_out=w, momentum_out=mom, workspace=space(lib, op))
    want = -iterate(1.5 * g)
    assert np.linalg.norm(w.get() - want) <= limit(t, want)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_norms_far_under_eps(lib, t):
    """X is u / eps then, and its elements small beside what singular values of 1 have."""
    m, n = 136, 200
    rng = np.random.default_rng(9)
    for ratio in (1e-2, 1e-4, 1e-6):
        v = rng.standard_normal((m, 8)) @ rng.standard_normal((8, n))
        v = R.unpack(R.pack(v * (1e-7 * ratio / np.linalg.norm(v)), t), t)
        o, op = Mat(lib, t, m, n), ops.Muon(m, n, t, exact=True)
        op.orthogonalize(Mat(lib, t, m, n, v), o, workspace=space(lib, op))
        want = iterate(v)
        assert np.linalg.norm(o.get() - want) <= limit(t, want), ratio


@pytest.mark.parametrize("style", ["packed", "odd"])
def test_bfloat16_held_in_two_numbers(lib, style):
    """Strides, a batch, in place: what the kernels of two numbers do to the type."""
    for k, (batch, m, n) in enumerate([(1, 1, 9), (2, 9, 1), (4, 17, 33), (3, 130, 70), (1, 97, 500), (2, 1000, 136)]):
        rng, L = np.random.default_rng(k), Layout(lib, "bf16", style)
        v = R.unpack(R.pack(rng.standard_normal((batch, m, n)), "bf16"), "bf16")
        u, o = L(batch * m, n, v.reshape(-1, n)), L(batch * m, n)
        op = ops.Muon(m, n, "bf16", batch=batch, ld_u=L.ld(n), ld_o=L.ld(n), exact=True)
        ws = space(lib, op)
        op.orthogonalize(u, o, workspace=ws)
        got = o.get().reshape(batch, m, n)
        for z in range(batch):
            want = iterate(v[z])  # of few values a rounding may be half a step of each
            assert np.linalg.norm(got[z] - want) <= (TWO + HALF["bf16"]) * np.linalg.norm(want)
        ws.check()
        before = o.bits()
        op.orthogonalize(u, u, workspace=ws)
        assert np.array_equal(u.bits(), before)
