"""The kernels of the operators' products (volta_amd/csrc/ops_gemm.h), tile by
tile: which plans they take, and their epilogues; and the layers at sizes whose
plans take each tile, whole and split."""
from __future__ import annotations

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import Mat, act, act_error, check, rounded
from tests.test_gpu_ops import GATED, LINEAR, NN, NT, SHAPES, STORE, TILES, TN, U32, Space, _forms, draws, sum_error, whole
from tests.test_ops import plan
from volta_amd import load_hip, ops

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


class Product:
    """Operands of whole numbers, as direct loads take them or not."""

    def __init__(self, lib, t, layout, kind, direct, M, K, N, rng):
        e = 16 // (4 if t == "f32" else 2)
        if direct:
            M, K, N = ((M + e - 1) // e * e if layout == TN else M, (K + e - 1) // e * e if layout != TN else K,
                       (N + e - 1) // e * e if layout != NT else N)
        self.lib, self.t, self.layout, self.kind, self.direct, self.dims = lib, t, layout, kind, direct, (M, K, N)
        self.pad, self.lead = (e, 0) if direct else (3, 1)
        self.P = whole(rng, M, K)
        self.Q = [whole(rng, K, N) for _ in range(2 if kind == GATED else 1)]
        self.p = self.mat(*((K, M, self.P.T) if layout == TN else (M, K, self.P)))
        self.q = [self.mat(*((N, K, v.T) if layout == NT else (K, N, v))) for v in self.Q]

    def mat(self, rows, cols, v=None, more=0):
        return Mat(self.lib, self.t, rows, cols, v, ld=cols + self.pad + more, lead=self.lead)

    def vec(self, v):
        return Mat(self.lib, self.t, 1, v.size, v, lead=self.lead)

    def sums(self):
        return [self.P @ v for v in self.Q]

    def run(self, tile, splits, out, act="identity", bias=(None, None), residual=None, pre=(None, None), unit=None):
        M, K, N = self.dims

        def at(m):
            return None if m is None else m.ptr

        rc = self.lib.lib.volta_hip_op_product_with(
            R.TYPES.index(self.t), self.layout, self.kind, TILES[tile], splits, int(self.direct), self.p.ptr, self.p.ptr,
            self.p.ld, self.q[0].ptr, self.q[-1].ptr, self.q[0].ld, out.ptr, out.ptr, out.ld, M, N, K, 1, 1, ops.ACTS[act],
            at(bias[0]), at(bias[1]), at(residual), residual.ld if residual else 0, at(pre[0]), at(pre[1]),
            pre[0].ld if pre[0] else 0, at(unit))
        assert rc == 0

    def same(self, m, want, what):
        """Equal to the last bit but for the sign of a zero."""
        got, want = m.get(), R.unpack(R.pack(want, self.t), self.t)
        bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
        assert not bad.any(), (what, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.filterwarnings("ignore:overflow encountered in cast")
def test_epilogues_on_every_tile(lib, t):
    """Bias, activation, residual (its own matrix, and in the output's place)
    and kept pre-activations of each tile and form of loads, whole and split
    over k, at sizes around the tiles' edges.  Whole numbers under 2^24 in 32
    bits, so the results are exact, rounded once."""
    for layout, kind, tile, direct in _forms(t):
        if kind == STORE:
            continue
        for n, (M, K, N) in enumerate(SHAPES):
            for splits in (1, 3):
                a = ("relu", "identity")[(n + splits) % 2]
                print(t, "kind", kind, "tile", tile, "direct", direct, M, K, N, "splits", splits, a, flush=True)
                rng = np.random.default_rng(2000 * n + splits)
                x = Product(lib, t, layout, kind, direct, M, K, N, rng)
                rows, cols = x.dims[0], x.dims[2]
                b = [rng.integers(-50, 51, cols).astype(np.float64) for _ in x.Q]
                r = rng.integers(-50, 51, (rows, cols)).astype(np.float64)
                bias, keep = [x.vec(v) for v in b], [x.mat(rows, cols, more=2 * x.pad) for _ in x.Q]
                p = [s + v for s, v in zip(x.sums(), b)]
                f = act(a, p[0])[0]
                out = x.mat(rows, cols)
                if kind == GATED:
                    x.run(tile, splits, out, a, bias, None, keep)
                    x.same(out, f * p[1], "h")
                    x.same(keep[1], p[1], "up")
                    one = x.mat(rows, cols)  # one bias, nothing kept
                    x.run(tile, splits, one, a, (None, bias[1]))
                    x.same(one, act(a, p[0] - b[0])[0] * p[1], "h without the gate's bias")
                else:
                    res = x.mat(rows, cols, r, more=x.pad)
                    x.run(tile, splits, out, a, (bias[0], None), res, (keep[0], None))
                    x.same(out, f + r, "y")
                    into = x.mat(rows, cols, r)
                    x.run(tile, splits, into, a, (None, None), into)
                    x.same(into, act(a, p[0] - b[0])[0] + r, "y in the residual's place")
                x.same(keep[0], p[0], "pre")


def test_units_on_every_tile(lib):
    """Sums in float16 in units of a power of two."""
    for layout, kind, tile, direct in _forms("f16"):
        if kind != STORE:
            continue
        for n, (M, K, N) in enumerate(SHAPES):
            for splits, unit in ((1, 2.0**-7), (3, 2.0**3)):
                print("layout", layout, "tile", tile, "direct", direct, M, K, N, "splits", splits, flush=True)
                x = Product(lib, "f16", layout, kind, direct, M, K, N, np.random.default_rng(3000 * n + splits))
                out = x.mat(x.dims[0], x.dims[2])
                x.run(tile, splits, out, unit=Mat(lib, "f32", 1, 1, np.array([[unit]])))
                x.same(out, x.sums()[0] * unit, "sums")


# (bytes of an element, gated): (tile, split over k, rows, inputs, outputs), the operands packed and
# aligned ("direct") or one element off ("staged")
PLANS = {
    (2, 0): {"direct": [(0, 0, 8200, 40, 1000), (0, 1, 1030, 8192, 1000), (1, 0, 5000, 40, 776), (2, 0, 8200, 40, 136),
                        (2, 1, 1030, 4096, 200), (3, 0, 8200, 40, 72), (3, 1, 513, 2048, 64), (4, 0, 513, 40, 64),
                        (4, 1, 17, 4096, 64), (5, 0, 1, 264, 64), (5, 1, 1, 8192, 64), (6, 0, 1, 40, 64),
                        (6, 1, 1, 4096, 64), (7, 0, 257, 40, 1000)],
             "staged": [(2, 0, 8200, 40, 72), (2, 1, 65, 8192, 1032), (4, 0, 513, 40, 64), (4, 1, 1, 4096, 64),
                        (5, 1, 1, 4096, 1032), (6, 1, 1, 8192, 64), (7, 0, 257, 40, 1000), (7, 1, 130, 8192, 136)]},
    (2, 1): {"direct": [(0, 0, 5000, 40, 776), (0, 1, 1000, 8192, 520), (1, 0, 8200, 40, 200), (2, 0, 8200, 40, 72),
                        (2, 1, 1030, 4096, 104), (3, 0, 4100, 40, 104), (3, 1, 1, 4096, 64), (4, 0, 513, 40, 64),
                        (4, 1, 3, 4096, 64), (5, 0, 1, 40, 64), (5, 1, 65, 4096, 72), (6, 0, 257, 40, 520),
                        (6, 1, 130, 4096, 104), (7, 0, 257, 40, 1000), (7, 1, 33, 4096, 520)],
             "staged": [(2, 0, 4100, 40, 104), (2, 1, 513, 8192, 264), (4, 0, 513, 40, 64), (4, 1, 1, 1504, 64),
                        (5, 1, 1, 2048, 1032), (6, 1, 257, 2048, 200), (7, 0, 257, 200, 1000), (7, 1, 300, 2048, 200)]},
    (4, 0): {"direct": [(0, 0, 8200, 40, 1000), (0, 1, 8200, 1032, 200), (1, 0, 5000, 40, 776), (1, 1, 1030, 4096, 72),
                        (2, 0, 8200, 40, 200), (2, 1, 1030, 1504, 72), (3, 0, 8200, 40, 72), (3, 1, 513, 1000, 72),
                        (4, 0, 513, 40, 64), (4, 1, 513, 520, 64), (5, 0, 1, 200, 64), (5, 1, 1, 4096, 64),
                        (6, 0, 1, 40, 64), (7, 0, 257, 40, 1000)],
             "staged": [(4, 0, 513, 40, 64), (4, 1, 513, 264, 64), (5, 1, 1, 2048, 64), (7, 0, 257, 40, 1000),
                        (7, 1, 200, 4096, 136)]},
    (4, 1): {"direct": [(0, 0, 5000, 40, 776), (0, 1, 8200, 1032, 104), (1, 0, 8200, 40, 200), (1, 1, 513, 4096, 264),
                        (2, 0, 1030, 40, 1000), (2, 1, 1030, 1000, 104), (3, 0, 4100, 40, 104), (3, 1, 513, 1000, 64),
                        (4, 0, 513, 40, 64), (4, 1, 513, 520, 64), (5, 0, 1, 40, 64), (5, 1, 1, 2048, 64),
                        (6, 0, 257, 40, 520), (7, 0, 257, 40, 1000)],
             "staged": [(4, 0, 513, 40, 64), (4, 1, 513, 264, 64), (5, 1, 1, 1000, 64), (6, 1, 257, 1504, 104),
                        (7, 0, 257, 40, 1000), (7, 1, 300, 8192, 136)]},
}


def _planned(e, kind, form, tile, split, M, K, N):
    got = plan(e, NN, kind, M, N, K, direct=int(form == "direct"))
    assert got[0] == tile and (got[1] > 1) == bool(split), ("the plan of this size is another one now", got)


@pytest.mark.parametrize("form", ["direct", "staged"])
@pytest.mark.parametrize("t", R.TYPES)
def test_linear_layers_on_every_tile(lib, t, form):
    """Bias, GELU, residual and kept pre-activations at sizes whose plans take
    each tile, whole and split."""
    e, lead = (4 if t == "f32" else 2), 0 if form == "direct" else 1
    for n, (tile, split, M, K, N) in enumerate(PLANS[e, 0][form]):
        print(t, form, "tile", tile, "split", split, M, K, N, flush=True)
        _planned(e, LINEAR, form, tile, split, M, K, N)
        rng = np.random.default_rng(700 + n)
        x, w = draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5)
        b, r = draws(rng, t, N), draws(rng, t, M, N)
        mx, mw, mb = Mat(lib, t, M, K, x, lead=lead), Mat(lib, t, K, N, w, lead=lead), Mat(lib, t, 1, N, b, lead=lead)
        mr, y, pre = (Mat(lib, t, M, N, v, ld=N + 8 * i, lead=lead) for i, v in ((1, r), (2, None), (3, None)))
        op = ops.Linear(M, K, N, t, "gelu", ld_residual=mr.ld, ld_y=y.ld, ld_pre=pre.ld)
        ws = Space(lib, op)
        op.forward(mx, mw, y, bias=mb, residual=mr, pre=pre, workspace=ws)
        p = x @ w + b
        ep = sum_error(x, w, K) + 2 * U32 * np.abs(p)
        want = act("gelu", p)[0] + r
        tol = 1.2 * ep + act_error(t, p)[0] + 2 * U32 * np.abs(want)
        check(y.get(), want, 1.01 * tol + rounded(want, t), "y")
        check(pre.get(), p, 1.01 * ep + rounded(p, t), "pre")
        into = Mat(lib, t, M, N, r, ld=mr.ld, lead=lead)
        ops.Linear(M, K, N, t, "gelu", ld_residual=mr.ld, ld_y=mr.ld).forward(mx, mw, into, bias=mb, residual=into,
                                                                             workspace=ws)
        assert np.array_equal(into.bits(), y.bits())
        ws.check()


@pytest.mark.parametrize("form", ["direct", "staged"])
@pytest.mark.parametrize("t", R.TYPES)
def test_gated_layers_on_every_tile(lib, t, form):
    e, lead = (4 if t == "f32" else 2), 0 if form == "direct" else 1
    for n, (tile, split, M, K, N) in enumerate(PLANS[e, 1][form]):
        print(t, form, "tile", tile, "split", split, M, K, N, flush=True)
        _planned(e, GATED, form, tile, split, M, K, N)
        rng = np.random.default_rng(800 + n)
        x, wg, wu = draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5), draws(rng, t, K, N, scale=K**-0.5)
        bg, bu = draws(rng, t, N), draws(rng, t, N)
        m = [Mat(lib, t, *v.shape, v, lead=lead) for v in (x, wg, wu)]
        vg, vu = (Mat(lib, t, 1, N, v, lead=lead) for v in (bg, bu))
        h, pg, pu = (Mat(lib, t, M, N, ld=N + 8 * i, lead=lead) for i in (1, 2, 2))
        op = ops.GatedFF(M, K, N, t, "silu", ld_h=h.ld, ld_pre=pg.ld)
        ws = Space(lib, op)
        op.forward(*m, h, b_gate=vg, b_up=vu, gate=pg, up=pu, workspace=ws)
        g, u = x @ wg + bg, x @ wu + bu
        eg, eu = sum_error(x, wg, K) + 2 * U32 * np.abs(g), sum_error(x, wu, K) + 2 * U32 * np.abs(u)
        f, _ = act("silu", g)
        ef = 1.2 * eg + act_error(t, g)[0] + U32 * np.abs(f)
        want = f * u
        tol = ef * (np.abs(u) + eu) + np.abs(f) * eu + 2 * U32 * np.abs(want) + 1e-37
        check(h.get(), want, 1.01 * tol + rounded(want, t), "h")
        check(pg.get(), g, 1.01 * eg + rounded(g, t), "gate")
        check(pu.get(), u, 1.01 * eu + rounded(u, t), "up")
        ws.check()


@pytest.mark.parametrize("t", R.TYPES)
def test_layers_laid_out_anew_exactly(lib, t):
    """Operands whose rows are not whole 16-byte chunks, copied into the
    workspace first: whole numbers, so products, gradients and what is kept are
    exact."""
    M, K, N = 1600, 1001, 1501
    e = 4 if t == "f32" else 2
    rng = np.random.default_rng(79)
    x, wg, wu = whole(rng, M, K), whole(rng, K, N), whole(rng, K, N)
    # a few small whole numbers, so that the gated layer's products of them stay exact
    dh = rng.integers(-1, 2, (M, N)) * (rng.random((M, N)) < 0.05)

    def exact(m, want):
        return np.array_equal(m.get(), R.unpack(R.pack(want, t), t))

    lin = ops.Linear(M, K, N, t)
    even = ops.Linear(M, 1008, 1504, t)
    assert lin.workspace_bytes() >= even.workspace_bytes() + (M * K + K * N) * e, "not laid out anew"
    ws, wsb = Space(lib, lin), Space(lib, lin, True)
    mx, mw, mdh = Mat(lib, t, M, K, x), Mat(lib, t, K, N, wg), Mat(lib, t, M, N, dh)
    y, dx, dw = Mat(lib, t, M, N), Mat(lib, t, M, K), Mat(lib, t, K, N)
    lin.forward(mx, mw, y, workspace=ws)
    lin.backward(mdh, mx, mw, dx=dx, dw=dw, workspace=wsb)
    ws.check()
    wsb.check()
    assert exact(y, x @ wg) and exact(dx, dh @ wg.T) and exact(dw, x.T @ dh)
    gat = ops.GatedFF(M, K, N, t, "relu")
    ws, wsb = Space(lib, gat), Space(lib, gat, True)
    mu, h, g, u = Mat(lib, t, K, N, wu), Mat(lib, t, M, N), Mat(lib, t, M, N), Mat(lib, t, M, N)
    gat.forward(mx, mw, mu, h, gate=g, up=u, workspace=ws)
    p = [x @ wg, x @ wu]
    with np.errstate(over="ignore"):
        assert exact(h, np.maximum(p[0], 0) * p[1])
    assert exact(g, p[0]) and exact(u, p[1])
    kept = [whole(rng, M, N), whole(rng, M, N)]
    pre = [Mat(lib, t, M, N, v) for v in kept]
    dg, du = Mat(lib, t, K, N), Mat(lib, t, K, N)
    gat.backward(mdh, mx, mw, mu, *pre, dx=dx, dw_gate=dg, dw_up=du, workspace=wsb)
    d = [dh * kept[1] * (kept[0] > 0), dh * np.maximum(kept[0], 0)]
    assert exact(dx, d[0] @ wg.T + d[1] @ wu.T) and exact(dg, x.T @ d[0]) and exact(du, x.T @ d[1])
    ws.check()
    wsb.check()
