"""Gradients of a mean of losses, whose rows have one dloss alike, and of far and
infinite ones, on the GPU (include/volta_ops.h, volta_amd.ops.CrossEntropy).

Tolerances, of the norm.  dz's rounding and the result's are independent, and of a
value in [2^e, 2^(e+1)) evenly over a step each is step^2 / 12 of its square at most,
2 HALF / sqrt(12) of the norm; together sqrt(2) of that, and a tenth more for chance
and for what 32 bits leave.  A dloss of every row that were rounded the same way
would be up to HALF off alone, 1.7 times one of the two."""
from __future__ import annotations

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_graph import Captured, put, spoil
from tests.ops_ref import HALF, TYPES, Mat
from tests.test_gpu_ops import STORE, Space, _forms, draws, say
from tests.test_gpu_ops_loss import Words
from tests.test_gpu_ops_tiles import SHAPES, Product
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return load_hip()


class Problem:
    """A call's matrices, its gradients in 64 bits."""

    def __init__(self, lib, t, M, K, C, dloss, seed=0, nolabel=0.0):
        rng = np.random.default_rng(seed)
        self.x, self.w = draws(rng, t, M, K), draws(rng, t, K, C, scale=0.25)
        self.labels = rng.integers(0, C, M)
        self.labels[rng.random(M) < nolabel] = -1
        self.dloss = np.asarray(dloss, np.float32)
        z = self.x @ self.w
        top = z.max(1, keepdims=True)
        lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0].astype(np.float32)
        p = np.exp(z - lse[:, None].astype(np.float64))
        has = self.labels >= 0
        p[np.arange(M)[has], self.labels[has]] -= 1
        self.dz = np.where(has[:, None], p * np.where(has, self.dloss, 0).astype(np.float64)[:, None], 0.0)
        self.op = ops.CrossEntropy(M, K, C, t)
        self.ws = Space(lib, self.op, True)
        self.given = (Mat(lib, t, M, K, self.x), Mat(lib, t, K, C, self.w), Words(lib, self.labels),
                      Mat(lib, "f32", 1, M, lse), Mat(lib, "f32", 1, M, self.dloss))
        self.out = {"dx": Mat(lib, t, M, K), "dw": Mat(lib, t, K, C), "db": Mat(lib, t, 1, C)}

    def want(self):
        return {"dx": self.dz @ self.w.T, "dw": self.x.T @ self.dz, "db": self.dz.sum(0)[None]}

    def run(self, stream=0):
        self.op.backward(*self.given, **self.out, workspace=self.ws, stream=stream)


def near(t, got, want, name):
    limit = 1.1 * np.sqrt(2) * 2 * HALF[t] / np.sqrt(12) * np.linalg.norm(want) + R.FLOOR[t] * np.sqrt(want.size)
    if t == "f32":  # sums in 32 bits
        limit = 1e-5 * np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= limit, (name, np.linalg.norm(got - want) / np.linalg.norm(want))


@pytest.mark.parametrize("rows", [1, 100, 128, 129, 255, 1020, 4080])
@pytest.mark.parametrize("t", TYPES)
def test_a_mean_over_rows(lib, t, rows):
    """1 / 255, 1 / 1020 and 1 / 4080 lie half a step from bfloat16's numbers."""
    p = Problem(lib, t, rows, 64, 4096, np.full(rows, 1 / rows))
    p.run()
    for name, want in p.want().items():
        near(t, p.out[name].get(), want, name)
    p.ws.check()


@pytest.mark.parametrize("t", TYPES)
def test_a_mean_over_rows_with_a_label(lib, t):
    """Rows without a label have a far larger dloss, which has no say."""
    p = Problem(lib, t, 600, 72, 1003, np.full(600, 1 / 510), nolabel=0.15)
    p.given[-1].dev = Mat(lib, "f32", 1, 600, np.where(p.labels < 0, 1e30, p.dloss)).dev
    p.given[-1].ptr = p.given[-1].dev.ptr
    p.run()
    for name, want in p.want().items():
        near(t, p.out[name].get(), want, name)


@pytest.mark.parametrize("scale", [2.0**-110, 1e-30, 1e-20, 1.0, 1e20, 1e34])
@pytest.mark.parametrize("rows", [96, 300])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_far_dloss(lib, t, rows, scale):
    p = Problem(lib, t, rows, 40, 500, np.full(rows, scale / rows))
    p.run()
    for name, want in p.want().items():
        assert np.abs(want).max() < 3e38
        near(t, p.out[name].get(), want, name)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("rows", [96, 300])
@pytest.mark.parametrize("t", TYPES)
def test_one_row_of_infinite_dloss(lib, t, rows, bad):
    """It reaches its own row of dx, and all of dw and db; the other rows keep their bits."""
    p = Problem(lib, t, rows, 40, 500, np.full(rows, 1e-5 / rows))
    want, d = p.want()["dx"], p.dloss.copy()
    d[7] = bad
    p.given[-1].dev = Mat(lib, "f32", 1, rows, d).dev
    p.given[-1].ptr = p.given[-1].dev.ptr
    p.run()
    got = p.out["dx"].get()
    assert not np.isfinite(got[7]).any() and not np.isfinite(p.out["db"].get()).any()
    near(t, np.delete(got, 7, 0), np.delete(want, 7, 0), "dx")


@pytest.mark.parametrize("t", TYPES)
def test_the_largest_of_many_rows(lib, t):
    """More rows than one block looks at; the largest dloss in the last one, and
    captured into a graph, on other values each time."""
    M = 150001
    d = np.full(M, 1e-4)
    d[-1] = 0.75
    p = Problem(lib, t, M, 8, 24, d)
    p.run()
    first = {n: m.bits() for n, m in p.out.items()}
    want = p.want()
    for name in ("dx", "dw"):
        near(t, p.out[name].get(), want[name], name)
    graph = Captured(lib, p.run)
    for scale in (1.0, 16.0, 2.0**-9):
        put(lib, p.given[-1], (d * scale)[None])
        for m in p.out.values():
            spoil(lib, m)
        graph.replay()
        if scale == 1.0:
            assert all(np.array_equal(m.bits(), first[n]) for n, m in p.out.items())
        if t != "f16":  # subnormal gradients are rounded otherwise
            assert all(np.array_equal(m.get(), R.unpack(first[n].view(R.STORE[t]), t) * scale) for n, m in p.out.items())
    graph.close()


def test_units_of_bfloat16_on_every_tile(lib):
    """Sums of whole numbers times a power of two: exact up to the result's rounding."""
    for layout, kind, tile, direct in _forms("bf16"):
        if kind != STORE:
            continue
        for n, (M, K, N) in enumerate(SHAPES):
            for splits, unit in ((1, 2.0**-7), (3, 2.0**3)):
                say("layout", layout, "tile", tile, "direct", direct, M, K, N, "splits", splits)
                x = Product(lib, "bf16", layout, kind, direct, M, K, N, np.random.default_rng(3000 * n + splits))
                out = x.mat(x.dims[0], x.dims[2])
                x.run(tile, splits, out, unit=Mat(lib, "f32", 1, 1, np.array([[unit]])))
                x.same(out, x.sums()[0] * unit, "sums")
