"""The feed-forward operators (include/volta_ops.h) on the GPU against their
definitions in 64 bits: products on every tile, the layers with their
epilogues and gradients, the norm, dropout; odd sizes, strides, rows of zero
length, graphs and streams.

Tolerances.  A sum of K products in 32 bits is off by at most (K + 2) 2^-24 of
the sum of the products' magnitudes, whatever its order; a result rounded to
its type by half a step of it (tests/ops_ref.py HALF); the activations by
act_error; an operand rounded to the type before a product by half a step of
it times the other factor."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import HALF, TYPES, Mat, act, act_error, check, rounded
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu

TILES = {"256": 0, "256x128": 1, "128": 2, "64x128": 3, "64": 4, "skinny16": 5, "skinny32": 6, "skinny64": 7}
NN, NT, TN = 0, 1, 2
LINEAR, GATED, STORE = 0, 1, 2
U32 = 2.0**-24


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def say(*a):
    print(*a, flush=True)


def whole(rng, *shape):
    """Small whole numbers: every product's sum is exact in 32 bits, in any order."""
    return rng.integers(-3, 4, shape).astype(np.float64)


class Space:
    """A workspace as the operators take it."""

    def __init__(self, lib, op, backward=False):
        n = op.workspace_bytes(backward=backward)
        self.mat = R.Mat(lib, "f32", 1, n // 4) if n else None
        self.ptr, self.nbytes = (self.mat.ptr, n) if n else (0, 0)

    def check(self):
        if self.mat:
            self.mat.bits()


# ---------------------------------------------------------------------------
# Products on every tile, exact.
# ---------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (5, 9, 3), (16, 64, 32), (17, 65, 33), (64, 128, 96), (65, 200, 100), (130, 72, 264),
          (257, 136, 520), (300, 520, 257)]


def _product(lib, t, layout, kind, tile, splits, direct, M, N, K, rng, pieces=1, outputs=1):
    e = 16 // (4 if t == "f32" else 2)
    pad = 3 if not direct else e  # rows longer than the matrix, unaligned unless the direct form needs them aligned

    def mat(rows, cols, v):
        return Mat(lib, t, rows, cols, v, ld=cols + pad, lead=0 if direct else 1)

    P = [whole(rng, M, K) for _ in range(pieces)]
    two = 2 if kind == GATED else max(outputs, pieces)
    Q = [whole(rng, K, N) for _ in range(two)]
    p = [mat(*((K, M, x.T) if layout == TN else (M, K, x))) for x in P]
    q = [mat(*((N, K, x.T) if layout == NT else (K, N, x))) for x in Q]
    n_out = outputs
    out = [Mat(lib, t, M, N, ld=N + pad, lead=0 if direct else 1) for _ in range(n_out)]
    rc = lib.lib.volta_hip_op_product(R.TYPES.index(t), layout, kind, tile, splits, int(direct), p[0].ptr, p[-1].ptr,
                                      p[0].ld, q[0].ptr, q[-1].ptr, q[0].ld, out[0].ptr, out[-1].ptr, out[0].ld, M, N,
                                      K, pieces, outputs)
    assert rc == 0
    if kind == GATED:
        g, u = P[0] @ Q[0], P[0] @ Q[1]
        f, _ = act("silu", g)
        want = f * u
        check(out[0].get(), R.held(want, t), rounded(want, t) * 1.001 + act_error(t, g)[0] * np.abs(u) + 1e-30,
              "gated product")
        return
    for z in range(n_out):
        want = sum(P[i] @ Q[i] for i in range(pieces)) if pieces > 1 else P[0] @ Q[z]
        got = out[z].bits().view(R.STORE[t])
        assert np.array_equal(got, R.pack(want, t)), f"output {z}"


def _forms(t):
    for layout, kinds in ((NN, (LINEAR, GATED)), (NT, (STORE,)), (TN, (STORE,))):
        for kind in kinds:
            for tile in TILES:
                for direct in (False, True):
                    if tile in ("256", "256x128", "64x128") and not direct:
                        continue
                    if tile.startswith("skinny") and layout == TN:
                        continue
                    yield layout, kind, tile, direct


@pytest.mark.parametrize("t", TYPES)
def test_products_on_every_tile(lib, t):
    """Every tile, layout and form of loads at sizes around its edges, whole
    and split over k: the sums are whole numbers, so the results are exact."""
    e = 16 // (4 if t == "f32" else 2)
    for layout, kind, tile, direct in _forms(t):
        for n, (M, K, N) in enumerate(SHAPES):
            if direct:
                M, K, N = ((M + e - 1) // e * e if layout == TN else M, (K + e - 1) // e * e if layout != TN else K,
                           (N + e - 1) // e * e if layout != NT else N)
            for splits in (1, 3):
                say(t, "layout", layout, "kind", kind, "tile", tile, "direct", direct, "M", M, "K", K, "N", N, "splits",
                    splits)
                rng = np.random.default_rng(1000 * n + splits)
                _product(lib, t, layout, kind, TILES[tile], splits, direct, M, N, K, rng,
                         pieces=2 if layout == NT and n % 2 else 1, outputs=2 if layout == TN and n % 2 else 1)


@pytest.mark.parametrize("t", TYPES)
def test_product_over_no_rows_is_zero(lib, t):
    _product(lib, t, TN, STORE, TILES["128"], 1, False, 40, 24, 0, np.random.default_rng(0), outputs=2)


# ---------------------------------------------------------------------------
# The layers.
# ---------------------------------------------------------------------------
class Layout:
    """How a test's matrices lie: packed, or in wider rows at odd elements."""

    def __init__(self, lib, t, style):
        self.lib, self.t, self.style = lib, t, style
        self.pad, self.lead = {"packed": (0, 0), "odd": (3, 1), "wide": (32, 16)}[style]

    def ld(self, cols):
        return cols + self.pad

    def __call__(self, rows, cols, v=None):
        return Mat(self.lib, self.t, rows, cols, v, ld=cols + self.pad, lead=self.lead)

    def vec(self, n, v=None):
        return Mat(self.lib, self.t, 1, n, v, lead=self.lead)


def draws(rng, t, *shape, scale=1.0):
    """Normal values as type t holds them."""
    return R.unpack(R.pack(scale * rng.standard_normal(shape), t), t)


LAYERS = [(1, 8, 8), (1, 1000, 300), (3, 1, 5), (16, 256, 512), (17, 65, 31), (50, 384, 100), (64, 1024, 64),
          (65, 40, 264), (200, 300, 130), (384, 512, 256), (0, 24, 16)]
STYLES = ["packed", "odd", "wide"]
ACTS = ["identity", "relu", "sigmoid", "tanh", "leaky_relu", "silu", "gelu"]


def sum_error(x, w, K):
    return (K + 2) * U32 * (np.abs(x) @ np.abs(w))


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_linear_forward(lib, t, style):
    for n, (M, K, N) in enumerate(LAYERS):
        a, rng, L = ACTS[n % len(ACTS)], np.random.default_rng(n), Layout(lib, t, style)
        bias, residual, keep = n % 2 == 0, n % 3 != 1, n % 3 != 2
        say(t, style, a, M, K, N, "bias", bias, "residual", residual, "pre", keep)
        x, w = draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5)
        b, r = draws(rng, t, N), draws(rng, t, M, N)
        dx, dw, db, dr, y, pre = L(M, K, x), L(K, N, w), L.vec(N, b), L(M, N, r), L(M, N), L(M, N)
        op = ops.Linear(M, K, N, t, a, ld_x=L.ld(K), ld_w=L.ld(N), ld_y=L.ld(N), ld_residual=L.ld(N), ld_pre=L.ld(N))
        ws = Space(lib, op)
        op.forward(dx, dw, y, bias=db if bias else None, residual=dr if residual else None, pre=pre if keep else None,
                   workspace=ws)
        p = x @ w + (b if bias else 0)
        ep = sum_error(x, w, K) + 2 * U32 * np.abs(p)
        f, slope = act(a, p)
        want = f + (r if residual else 0)
        tol = 1.2 * ep + (act_error(t, p)[0] if a not in ("identity", "relu") else 0) + 2 * U32 * np.abs(want)
        check(y.get(), want, 1.01 * tol + rounded(want, t), "y")
        if keep:
            check(pre.get(), p, 1.01 * ep + rounded(p, t), "pre")
        else:
            assert pre.untouched()
        ws.check()
        if residual and M:  # the residual in y's place
            before = y.bits()
            op.forward(dx, dw, dr, bias=db if bias else None, residual=dr, workspace=ws)
            assert np.array_equal(dr.bits(), before)


def _backward_tol(t, x, d, ed, K, want):
    """Of x^T d or d w^T: d is off by ed and rounded to the type."""
    return np.abs(x) @ (ed + rounded(d, t)) * 1.001 + sum_error(x, np.abs(d) + ed, K) + rounded(want, t) * 1.01


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_linear_backward(lib, t, style):
    for n, (M, K, N) in enumerate(LAYERS):
        a, rng, L = ACTS[n % len(ACTS)], np.random.default_rng(50 + n), Layout(lib, t, style)
        say(t, style, a, M, K, N)
        x, w, dy, p = (draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5), draws(rng, t, M, N, scale=0.1),
                       draws(rng, t, M, N))
        op = ops.Linear(M, K, N, t, a, ld_x=L.ld(K), ld_w=L.ld(N), ld_y=L.ld(N), ld_pre=L.ld(N), ld_dx=L.ld(K),
                        ld_dw=L.ld(N))
        ws = Space(lib, op, True)
        mx, mw, mdy, mp = L(M, K, x), L(K, N, w), L(M, N, dy), L(M, N, p)
        dx, dw, db = L(M, K), L(K, N), L.vec(N)
        op.backward(mdy, mx, mw, pre=mp, dx=dx, dw=dw, db=db, workspace=ws)
        _, slope = act(a, p)
        d = dy * slope
        ed = np.abs(dy) * (act_error(t, p)[1] if a not in ("identity", "relu", "leaky_relu") else 0) + 2 * U32 * np.abs(d)
        want = d @ w.T
        if a == "identity":  # dy itself is the operand: no rounding before the products
            tol_dx = sum_error(d, w.T, N) + rounded(want, t)
            tol_dw = sum_error(x.T, d, M) + rounded(x.T @ d, t)
        else:
            tol_dx = _backward_tol(t, w, d.T, ed.T, N, want.T).T
            tol_dw = _backward_tol(t, x.T, d, ed, M, x.T @ d)
        check(dx.get(), want, tol_dx * 1.001 + 1e-37, "dx")
        check(dw.get(), x.T @ d, tol_dw * 1.001 + 1e-37, "dw")
        want = d.sum(0)[None]
        check(db.get(), want, (ed.sum(0) + (M + 2) * U32 * np.abs(d).sum(0))[None] + rounded(want, t) * 1.01 + 1e-37, "db")
        ws.check()
        # each gradient alone, the same bits
        for name, m in (("dx", dx), ("dw", dw), ("db", db)):
            again = L(m.rows, m.cols)
            op.backward(mdy, mx, mw, pre=mp, workspace=ws, **{name: again})
            assert np.array_equal(again.bits(), m.bits()), name


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_gated_forward(lib, t, style):
    for n, (M, K, N) in enumerate(LAYERS):
        a, rng, L = ACTS[(n + 5) % len(ACTS)], np.random.default_rng(100 + n), Layout(lib, t, style)
        bias, keep = n % 2 == 1, n % 3 != 0
        say(t, style, a, M, K, N, "bias", bias, "pre", keep)
        x, wg, wu = draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5), draws(rng, t, K, N, scale=K**-0.5)
        bg, bu = draws(rng, t, N), draws(rng, t, N)
        op = ops.GatedFF(M, K, N, t, a, ld_x=L.ld(K), ld_w=L.ld(N), ld_h=L.ld(N), ld_pre=L.ld(N))
        ws = Space(lib, op)
        h, pg, pu = L(M, N), L(M, N), L(M, N)
        op.forward(L(M, K, x), L(K, N, wg), L(K, N, wu), h, b_gate=L.vec(N, bg) if bias else None,
                   b_up=L.vec(N, bu) if bias else None, gate=pg if keep else None, up=pu if keep else None, workspace=ws)
        g, u = x @ wg + (bg if bias else 0), x @ wu + (bu if bias else 0)
        eg, eu = sum_error(x, wg, K) + 2 * U32 * np.abs(g), sum_error(x, wu, K) + 2 * U32 * np.abs(u)
        f, _ = act(a, g)
        ef = 1.2 * eg + (act_error(t, g)[0] if a not in ("identity", "relu") else 0) + U32 * np.abs(f)
        want = f * u
        tol = ef * (np.abs(u) + eu) + np.abs(f) * eu + 2 * U32 * np.abs(want) + 1e-37
        check(h.get(), want, 1.01 * tol + rounded(want, t), "h")
        if keep:
            check(pg.get(), g, 1.01 * eg + rounded(g, t), "gate")
            check(pu.get(), u, 1.01 * eu + rounded(u, t), "up")
        ws.check()


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_gated_backward(lib, t, style):
    for n, (M, K, N) in enumerate(LAYERS):
        a, rng, L = ACTS[(n + 4) % len(ACTS)], np.random.default_rng(150 + n), Layout(lib, t, style)
        say(t, style, a, M, K, N)
        x, wg, wu = draws(rng, t, M, K), draws(rng, t, K, N, scale=K**-0.5), draws(rng, t, K, N, scale=K**-0.5)
        dh, g, u = draws(rng, t, M, N, scale=0.1), draws(rng, t, M, N), draws(rng, t, M, N)
        op = ops.GatedFF(M, K, N, t, a, ld_x=L.ld(K), ld_w=L.ld(N), ld_h=L.ld(N), ld_pre=L.ld(N), ld_dx=L.ld(K),
                         ld_dw=L.ld(N))
        ws = Space(lib, op, True)
        args = (L(M, N, dh), L(M, K, x), L(K, N, wg), L(K, N, wu), L(M, N, g), L(M, N, u))
        out = {"dx": L(M, K), "dw_gate": L(K, N), "dw_up": L(K, N), "db_gate": L.vec(N), "db_up": L.vec(N)}
        op.backward(*args, workspace=ws, **out)
        f, slope = act(a, g)
        inexact = a not in ("identity", "relu", "leaky_relu")
        ef, es = act_error(t, g) if inexact else (0, 0)
        dg, du = dh * u * slope, dh * f
        eg = np.abs(dh * u) * es + 3 * U32 * np.abs(dg)
        eu = np.abs(dh) * ef + 2 * U32 * np.abs(du) + U32 * np.abs(du)
        want = dg @ wg.T + du @ wu.T
        cat, ecat, wcat = np.hstack([dg, du]), np.hstack([eg, eu]), np.hstack([wg, wu])
        check(out["dx"].get(), want, _backward_tol(t, wcat, cat.T, ecat.T, 2 * N, want.T).T + 1e-37, "dx")
        for name, d, ed in (("gate", dg, eg), ("up", du, eu)):
            want = x.T @ d
            check(out["dw_" + name].get(), want, _backward_tol(t, x.T, d, ed, M, want) + 1e-37, "dw_" + name)
            want = d.sum(0)[None]
            check(out["db_" + name].get(), want,
                  (ed.sum(0) + (M + 2) * U32 * np.abs(d).sum(0))[None] * 1.01 + rounded(want, t) * 1.01 + 1e-37,
                  "db_" + name)
        ws.check()
        for some in (["dx"], ["dw_gate", "dw_up"], ["db_gate"], ["db_up"]):
            again = {k: L(out[k].rows, out[k].cols) for k in some}
            op.backward(*args, workspace=ws, **again)
            for k in some:
                assert np.array_equal(again[k].bits(), out[k].bits()), k


@pytest.mark.parametrize("t", TYPES)
def test_gated_halves_of_one_matrix(lib, t):
    """Wg | Wu, gate | up and their gradients as the halves of wider matrices."""
    M, K, N = 40, 64, 48
    rng = np.random.default_rng(7)
    x, wg, wu, dh = draws(rng, t, M, K), draws(rng, t, K, N), draws(rng, t, K, N), draws(rng, t, M, N)
    size = 4 if t == "f32" else 2

    def half(m):
        return m.ptr + N * size

    plain = ops.GatedFF(M, K, N, t)
    both = ops.GatedFF(M, K, N, t, ld_w=2 * N, ld_pre=2 * N, ld_dw=2 * N)
    ws, wsb = Space(lib, plain), Space(lib, plain, True)
    mx, mdh, m1, m2 = Mat(lib, t, M, K, x), Mat(lib, t, M, N, dh), Mat(lib, t, K, N, wg), Mat(lib, t, K, N, wu)
    w = Mat(lib, t, K, 2 * N, np.hstack([wg, wu]))
    h1, h2, g, u = (Mat(lib, t, M, N) for _ in range(4))
    pre = Mat(lib, t, M, 2 * N)
    plain.forward(mx, m1, m2, h1, gate=g, up=u, workspace=ws)
    both.forward(mx, w.ptr, half(w), h2, gate=pre.ptr, up=half(pre), workspace=ws)
    assert np.array_equal(h1.bits(), h2.bits())
    assert np.array_equal(np.hstack([g.bits(), u.bits()]), pre.bits())
    d1, d2, dw = Mat(lib, t, K, N), Mat(lib, t, K, N), Mat(lib, t, K, 2 * N)
    plain.backward(mdh, mx, m1, m2, g, u, dw_gate=d1, dw_up=d2, workspace=wsb)
    both.backward(mdh, mx, w.ptr, half(w), pre.ptr, half(pre), dw_gate=dw.ptr, dw_up=half(dw), workspace=wsb)
    assert np.array_equal(np.hstack([d1.bits(), d2.bits()]), dw.bits())


@pytest.mark.parametrize("t", TYPES)
def test_operands_laid_out_anew(lib, t):
    """Products large enough that rows which are not whole 16-byte chunks are
    copied into the workspace first: the same values as through packed, aligned
    matrices of padded width, bit for bit where the padding is zeros."""
    M, K, N = 1600, 1001, 1501
    Kp, Np = 1008, 1504
    rng = np.random.default_rng(77)
    x, wg, wu, dh = draws(rng, t, M, K), draws(rng, t, K, N), draws(rng, t, K, N), draws(rng, t, M, N)

    def pad(v, r, c):
        out = np.zeros((r, c))
        out[: v.shape[0], : v.shape[1]] = v
        return out

    def run(op, lift, M, K, N):
        ws, wsb = Space(lib, op), Space(lib, op, True)
        m = {k: lift(r, c, v) for k, (r, c, v) in {"x": (M, K, x), "wg": (K, N, wg), "wu": (K, N, wu),
                                                   "dh": (M, N, dh)}.items()}
        o = {k: lift(r, c, None) for k, (r, c) in {"h": (M, N), "g": (M, N), "u": (M, N), "dx": (M, K), "dg": (K, N),
                                                   "du": (K, N)}.items()}
        if isinstance(op, ops.GatedFF):
            op.forward(m["x"], m["wg"], m["wu"], o["h"], gate=o["g"], up=o["u"], workspace=ws)
            op.backward(m["dh"], m["x"], m["wg"], m["wu"], o["g"], o["u"], dx=o["dx"], dw_gate=o["dg"], dw_up=o["du"],
                        workspace=wsb)
        else:
            op.forward(m["x"], m["wg"], o["h"], workspace=ws)
            op.backward(m["dh"], m["x"], m["wg"], dx=o["dx"], dw=o["dg"], workspace=wsb)
        ws.check()
        wsb.check()
        return {k: v.get() for k, v in o.items() if not v.untouched()}, (ws, wsb)

    e = 4 if t == "f32" else 2
    for make in (ops.GatedFF, ops.Linear):
        odd = make(M, K, N, t)
        even = make(M, Kp, Np, t)
        assert odd.workspace_bytes(backward=True) >= even.workspace_bytes(backward=True) + K * Np * e, "not laid out anew"
        got, _ = run(odd, lambda r, c, v: Mat(lib, t, r, c, v, lead=1), M, K, N)
        want, _ = run(even, lambda r, c, v: Mat(lib, t, r, c, None if v is None else pad(v, r, c)), M, Kp, Np)
        for k, v in got.items():
            w = want[k][: v.shape[0], : v.shape[1]]
            # a plan may split the sum elsewhere for the other size: equal but for the last rounding
            tol = rounded(w, t) * 2 + 4 * (Np + 2) * U32 * np.abs(w).max()
            check(v, w, tol, k)


# ---------------------------------------------------------------------------
# The norm.
# ---------------------------------------------------------------------------
NORMS = [(1, 1), (1, 4096), (3, 7), (5, 129), (9, 512), (4, 1000), (6, 1023), (3, 2056), (2, 5001), (2, 9000),
         (2, 17000), (1, 34001), (700, 72), (0, 64)]
EPS = 1e-6


def norm_ref(x, w, eps=EPS):
    rstd = 1 / np.sqrt((x**2).mean(1) + eps)
    return rstd, x * rstd[:, None] * w


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_norm_forward(lib, t, style):
    for n, (M, D) in enumerate(NORMS):
        rng, L = np.random.default_rng(200 + n), Layout(lib, t, style)
        residual, weight = n % 2 == 0, n % 3 != 2
        say(t, style, M, D, "residual", residual, "weight", weight)
        x, r, w = draws(rng, t, M, D), draws(rng, t, M, D, scale=3), draws(rng, t, D)
        op = ops.RmsNorm(M, D, t, EPS, ld_x=L.ld(D), ld_residual=L.ld(D), ld_sum=L.ld(D), ld_y=L.ld(D))
        mx, mr, mw, y, s, rstd = L(M, D, x), L(M, D, r), L.vec(D, w), L(M, D), L(M, D), R.floats(lib, M)
        kw = dict(weight=mw if weight else None, residual=mr if residual else None)
        op.forward(mx, y, sum=s, rstd=rstd, **kw)
        v = x + r if residual else x
        want_r, want = norm_ref(v, w if weight else 1.0)
        # the sum of D squares of values off by 2^-24 each; root, reciprocal
        rel = (D / 2 + 8) * U32
        check(s.get(), v, rounded(v, t) + U32 * np.abs(v), "sum")
        check(y.get(), want, (rel + 4 * U32) * np.abs(want) + rounded(want, t) * 1.01, "y")
        if M:
            check(rstd.get()[0], want_r, rel * want_r, "rstd")
        # s in the residual's or x's place, and nothing kept
        y2, into = L(M, D), mr if residual else mx
        op.forward(mx, y2, sum=into, **kw)
        assert np.array_equal(y2.bits(), y.bits()) and np.array_equal(into.bits(), s.bits())


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_norm_e4m3(lib, t, style, group):
    for n, (M, D) in enumerate(NORMS):
        rng, L = np.random.default_rng(250 + n), Layout(lib, t, style)
        say(t, style, M, D, "group", group)
        x, r, w = draws(rng, t, M, D), draws(rng, t, M, D, scale=3), draws(rng, t, D)
        if M > 1:
            x[1] = r[1] = 0  # a row of zeros has the smallest scale
        groups = -(-D // group) if group else 1
        op = ops.RmsNorm(M, D, t, EPS, out="e4m3", group=group, ld_x=L.ld(D), ld_residual=L.ld(D), ld_sum=L.ld(D),
                         ld_y=D + L.pad)
        y, s, scales = Mat(lib, "e4m3", M, D, ld=D + L.pad, lead=L.lead), L(M, D), Mat(lib, "f32", max(M, 1), groups)
        op.forward(L(M, D, x), y, weight=L.vec(D, w), residual=L(M, D, r), sum=s, scales=scales)
        if not M:
            assert y.untouched() and scales.untouched()
            continue
        _, v = norm_ref(x + r, w)
        rel = (D / 2 + 16) * U32
        got, sc = y.get(), scales.get()
        step = group or D
        for j in range(groups):
            c = slice(j * step, min(D, (j + 1) * step))
            want = np.maximum(np.abs(v[:, c]).max(1) / 448, 2.0**-126)
            check(sc[:, j], want, rel * want, "scales")
            # a code is off by half a step of it: of values up to 448 in units of the scale
            q = v[:, c] / sc[:, j:j + 1]
            check(got[:, c], q, rounded(q, "e4m3") * (1 + 2.0**-10) + rel * np.abs(q), "codes")
        check(s.get(), x + r, rounded(x + r, t) + U32 * np.abs(x + r), "sum")


@pytest.mark.parametrize("t", TYPES)
def test_norm_of_infinities_and_nan(lib, t):
    """A NaN or infinity spoils its own row, and in 8 bits its own groups' scales."""
    M, D = 5, 300
    rng = np.random.default_rng(3)
    x = draws(rng, t, M, D)
    clean = x.copy()
    x[1, 7], x[3, 299] = np.nan, np.inf
    y = Mat(lib, t, M, D)
    ops.RmsNorm(M, D, t, EPS).forward(Mat(lib, t, M, D, x), y)
    got = y.get()
    _, want = norm_ref(clean, 1.0)
    check(got[[0, 2, 4]], want[[0, 2, 4]], 200 * U32 * np.abs(want[[0, 2, 4]]) + rounded(want[[0, 2, 4]], t) * 1.01, "y")
    assert np.isnan(got[1]).all() and np.isnan(got[3, 299]) and (got[3, :299] == 0).all()
    c, sc = Mat(lib, "e4m3", M, D), Mat(lib, "f32", M, 3)
    ops.RmsNorm(M, D, t, EPS, out="e4m3", group=128).forward(Mat(lib, t, M, D, x), c, scales=sc)
    codes, scales = c.get(), sc.get()
    assert np.isnan(scales[1]).all() and np.isnan(codes[1]).all()
    assert np.isnan(scales[3, 2]) and np.isnan(codes[3, 256:]).all()
    assert (scales[3, :2] == 2.0**-126).all() and (codes[3, :256] == 0).all()
    assert np.isfinite(scales[[0, 2, 4]]).all() and np.isfinite(codes[[0, 2, 4]]).all()


@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_norm_backward(lib, t, style):
    for n, (M, D) in enumerate(NORMS + [(1500, 40), (600, 2100)]):
        rng, L = np.random.default_rng(300 + n), Layout(lib, t, style)
        add, weight = n % 2 == 0, n % 3 != 2
        say(t, style, M, D, "dsum", add, "weight", weight)
        dy, s, ds, w = draws(rng, t, M, D, scale=0.1), draws(rng, t, M, D), draws(rng, t, M, D, scale=0.1), draws(rng, t, D)
        rstd32 = (1 / np.sqrt((s**2).mean(1) + EPS)).astype(np.float32) if M else np.zeros(1, np.float32)
        rstd = rstd32.astype(np.float64)[:M, None]
        op = ops.RmsNorm(M, D, t, EPS, ld_x=L.ld(D), ld_sum=L.ld(D), ld_y=L.ld(D), ld_dx=L.ld(D))
        ws = Space(lib, op, True)
        mr = Mat(lib, "f32", 1, max(M, 1), rstd32[None])
        args = (L(M, D, dy), L(M, D, s), mr)
        mds, mw = L(M, D, ds), L.vec(D, w)
        kw = dict(weight=mw if weight else None, dsum=mds if add else None)
        dx, dw = L(M, D), L.vec(D)
        op.backward(*args, dx=dx, dweight=dw, workspace=ws, **kw)
        wv = w if weight else 1.0
        a, b = wv * dy * rstd, s * rstd**3
        c = (wv * dy * s).mean(1, keepdims=True)
        ec = (D + 6) * U32 * np.abs(wv * dy * s).mean(1, keepdims=True)
        want = a - b * c + (ds if add else 0)
        tol = 4 * U32 * np.abs(a) + np.abs(b) * (ec + 8 * U32 * np.abs(c)) + 3 * U32 * np.abs(want)
        check(dx.get(), want, 1.01 * tol + rounded(want, t) * 1.01, "dx")
        want = (dy * s * rstd).sum(0)[None]
        tol = (M + 4) * U32 * np.abs(dy * s * rstd).sum(0)[None]
        check(dw.get(), want, 1.01 * tol + rounded(want, t) * 1.01, "dweight")
        ws.check()
        dw2, dx2 = L.vec(D), L(M, D)
        op.backward(*args, dweight=dw2, workspace=ws, **kw)
        op.backward(*args, dx=dx2, **kw)
        assert np.array_equal(dw2.bits(), dw.bits()) and np.array_equal(dx2.bits(), dx.bits())
        if add:  # dx in dsum's place
            op.backward(*args, dx=mds, **kw)
            assert np.array_equal(mds.bits(), dx.bits())


# ---------------------------------------------------------------------------
# Dropout.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("style", STYLES)
@pytest.mark.parametrize("t", TYPES)
def test_dropout(lib, t, style):
    big = (1 << 64) - 5
    for n, (M, D, p, seed, offset) in enumerate([(1, 1, 0.5, 0, 0), (3, 7, 0.1, 1, 5), (5, 33, 0.3, big, big),
                                                 (4, 64, 0.0, 9, 0), (7, 130, 0.999, 4, 1 << 40), (0, 8, 0.5, 1, 1)]):
        rng, L = np.random.default_rng(400 + n), Layout(lib, t, style)
        residual = n % 2 == 1
        say(t, style, M, D, p)
        x, r = draws(rng, t, M, D), draws(rng, t, M, D)
        keep = R.splitmix_keep(M * D, seed, offset, p).reshape(M, D)
        if M > 2:
            x[~keep] = np.inf  # what is dropped does not reach y
        op = ops.Dropout(M, D, t, p, ld_x=L.ld(D), ld_residual=L.ld(D), ld_y=L.ld(D))
        mx, mr, y = L(M, D, x), L(M, D, r), L(M, D)
        op.forward(mx, y, residual=mr if residual else None, seed=seed, offset=offset)
        v = np.where(keep, np.where(keep, x, 0) / (1 - p), 0)
        want = v + (r if residual else 0)
        check(y.get(), want, 3 * U32 * (np.abs(v) + np.abs(want)) + rounded(want, t) * 1.01, "y")
        if M:
            into = mr if residual else mx  # in place
            op.forward(mx, into, residual=mr if residual else None, seed=seed, offset=offset)
            assert np.array_equal(into.bits(), y.bits())
            dx = L(M, D)
            op.backward(L(M, D, np.ones((M, D))), dx, seed=seed, offset=offset)
            assert np.array_equal(dx.get() != 0, keep)


def test_dropout_share(lib):
    """The share kept over a million elements is 1 - p within five deviations, and two offsets' masks agree by chance alone."""
    n, p = 1 << 20, 0.2
    one, out = Mat(lib, "f32", 1, n, np.ones((1, n))), Mat(lib, "f32", 1, n)
    op = ops.Dropout(1, n, "f32", p)
    masks = []
    for seed, offset in ((1, 0), (1, n // 2), (2, 0)):
        op.forward(one, out, seed=seed, offset=offset)
        masks.append(out.get()[0] != 0)
        assert abs(masks[-1].mean() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) ** 2
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs((masks[a] == masks[b]).mean() - agree) < 5 * (agree * (1 - agree) / n) ** 0.5


# ---------------------------------------------------------------------------
# Together: a residual block, forward and backward, against 64 bits and
# against differences; streams and captured graphs.
# ---------------------------------------------------------------------------
class Block:
    """y = s + dropout(gated(norm(s)) Wd), s = x + r, as a program keeps it."""

    def __init__(self, lib, t, M, D, H, p=0.25, seed=11):
        self.lib, self.t, self.dims, self.p, self.seed = lib, t, (M, D, H), p, seed
        rng = np.random.default_rng(5)
        self.v = {"x": draws(rng, t, M, D), "r": draws(rng, t, M, D), "wn": 1 + draws(rng, t, D, scale=0.1),
                  "wg": draws(rng, t, D, H, scale=D**-0.5), "wu": draws(rng, t, D, H, scale=D**-0.5),
                  "wd": draws(rng, t, H, D, scale=H**-0.5), "dy": draws(rng, t, M, D)}
        self.v["wn"] = R.unpack(R.pack(self.v["wn"], t), t)
        self.m = {k: Mat(lib, t, *(v.shape if v.ndim == 2 else (1, v.size)), v) for k, v in self.v.items()}
        for k, s in {"s": (M, D), "n": (M, D), "g": (M, H), "u": (M, H), "h": (M, H), "o": (M, D), "y": (M, D),
                     "do": (M, D), "dh": (M, H), "dn": (M, D), "dx": (M, D), "dwn": (1, D), "dwg": (D, H),
                     "dwu": (D, H), "dwd": (H, D)}.items():
            self.m[k] = Mat(lib, t, *s)
        self.m["rstd"] = Mat(lib, "f32", 1, M)
        self.norm, self.gated = ops.RmsNorm(M, D, t, EPS), ops.GatedFF(M, D, H, t)
        self.down, self.drop = ops.Linear(M, H, D, t), ops.Dropout(M, D, t, p)
        n = max(o.workspace_bytes(backward=b) for o in (self.norm, self.gated, self.down) for b in (False, True))
        self.ws = Mat(lib, "f32", 1, n // 4 + 4)
        self.ws.nbytes = n

    def run(self, stream=0):
        m, ws = self.m, self.ws
        kw = dict(workspace=ws, stream=stream)
        self.norm.forward(m["x"], m["n"], weight=m["wn"], residual=m["r"], sum=m["s"], rstd=m["rstd"], stream=stream)
        self.gated.forward(m["n"], m["wg"], m["wu"], m["h"], gate=m["g"], up=m["u"], **kw)
        self.down.forward(m["h"], m["wd"], m["o"], **kw)
        self.drop.forward(m["o"], m["y"], residual=m["s"], seed=self.seed, offset=3, stream=stream)
        self.drop.backward(m["dy"], m["do"], seed=self.seed, offset=3, stream=stream)
        self.down.backward(m["do"], m["h"], m["wd"], dx=m["dh"], dw=m["dwd"], **kw)
        self.gated.backward(m["dh"], m["n"], m["wg"], m["wu"], m["g"], m["u"], dx=m["dn"], dw_gate=m["dwg"],
                            dw_up=m["dwu"], **kw)
        self.norm.backward(m["dn"], m["s"], m["rstd"], m["dx"], weight=m["wn"], dsum=m["dy"], dweight=m["dwn"], **kw)

    OUT = ("y", "dx", "dwn", "dwg", "dwu", "dwd")

    def bits(self):
        return {k: self.m[k].bits() for k in self.OUT}

    def forward64(self, **v):
        v = {**self.v, **v}
        s = v["x"] + v["r"]
        _, n = norm_ref(s, v["wn"])
        g, u = n @ v["wg"], n @ v["wu"]
        h = act("silu", g)[0] * u
        keep = R.splitmix_keep(s.size, self.seed, 3, self.p).reshape(s.shape)
        return s + h @ v["wd"] * keep / (1 - self.p), (s, n, g, u, h, keep)


def test_block_gradients_against_differences(lib):
    """In float32, the directional derivative of sum(y dy) along each input is
    what central differences of the 64-bit block give (step 1e-5: their error
    is 1e-10 of the third derivative, and the products' sums 1e-5 of the
    magnitudes)."""
    b = Block(lib, "f32", 24, 40, 56)
    b.run()
    rng = np.random.default_rng(9)
    y, _ = b.forward64()
    check(b.m["y"].get(), y, 2e-5 * (1 + np.abs(y)), "y")
    for name, grad in (("x", "dx"), ("r", "dx"), ("wn", "dwn"), ("wg", "dwg"), ("wu", "dwu"), ("wd", "dwd")):
        v = rng.standard_normal(b.v[name].shape)
        eps = 1e-5
        up, dn = (b.forward64(**{name: b.v[name] + e * v})[0] for e in (eps, -eps))
        want = ((up - dn) * b.v["dy"]).sum() / (2 * eps)
        g = b.m[grad].get().reshape(v.shape)
        assert abs((g * v).sum() - want) <= 2e-5 * (np.abs(g) * np.abs(v)).sum() + 1e-6, name


@pytest.mark.parametrize("t", TYPES)
def test_block_against_64_bits(lib, t):
    """The whole block: every tensor between two operators is rounded to the
    type, so an output is off by a few half steps of its norm (eight roundings
    in a chain, none amplified by more than the block's gain of about 2)."""
    b = Block(lib, t, 70, 96, 200)
    b.run()
    y, (s, n, g, u, h, keep) = b.forward64()
    do = b.v["dy"] * keep / (1 - b.p)
    dh = do @ b.v["wd"].T
    f, slope = act("silu", g)
    dg, du = dh * u * slope, dh * f
    dn = dg @ b.v["wg"].T + du @ b.v["wu"].T
    rstd = 1 / np.sqrt((s**2).mean(1, keepdims=True) + EPS)
    d = dn * b.v["wn"]
    dx = rstd * d - s * rstd**3 * (d * s).mean(1, keepdims=True) + b.v["dy"]
    want = {"y": y, "dx": dx, "dwn": (dn * s * rstd).sum(0)[None], "dwg": n.T @ dg, "dwu": n.T @ du, "dwd": h.T @ do}
    for k, w in want.items():
        off = np.linalg.norm(b.m[k].get() - w) / np.linalg.norm(w)
        assert off <= 16 * HALF[t], (k, off)


def _hip(lib):
    """The HIP runtime the library runs on."""
    h = lib.lib
    for n, args in {"hipStreamCreate": [C.POINTER(C.c_void_p)], "hipStreamDestroy": [C.c_void_p],
                    "hipStreamSynchronize": [C.c_void_p], "hipStreamBeginCapture": [C.c_void_p, C.c_int],
                    "hipStreamEndCapture": [C.c_void_p, C.POINTER(C.c_void_p)],
                    "hipGraphInstantiate": [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t],
                    "hipGraphLaunch": [C.c_void_p, C.c_void_p], "hipGraphExecDestroy": [C.c_void_p],
                    "hipGraphDestroy": [C.c_void_p], "hipDeviceSynchronize": []}.items():
        fn = getattr(h, n)
        fn.restype, fn.argtypes = C.c_int, args
    return h


def test_block_on_a_stream_and_in_a_graph(lib):
    """The block on a stream of its own and replayed from a graph, eager runs
    between the replays: the same bits every time."""
    hip = _hip(lib)
    b, other = Block(lib, "bf16", 130, 256, 512), Block(lib, "bf16", 130, 256, 512, seed=12)
    b.run()
    other.run()
    want, other_want = b.bits(), other.bits()
    st = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(st)) == 0
    b.run(stream=st.value)
    assert hip.hipStreamSynchronize(st) == 0
    assert all(np.array_equal(v, want[k]) for k, v in b.bits().items())
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(st, 1) == 0  # thread-local
    b.run(stream=st.value)
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
    for _ in range(4):
        for k in Block.OUT:  # spoil the last replay's outputs
            m = b.m[k]
            lib.lib.volta_hip_copy(m.dev.ptr, m.before.ctypes.data, m.before.nbytes, 1)
        other.run()
        assert hip.hipDeviceSynchronize() == 0
        assert hip.hipGraphLaunch(run, st) == 0
        assert hip.hipStreamSynchronize(st) == 0
        assert all(np.array_equal(v, want[k]) for k, v in b.bits().items())
        assert all(np.array_equal(v, other_want[k]) for k, v in other.bits().items())
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    assert hip.hipStreamDestroy(st) == 0


def test_rows_far_into_a_large_matrix(lib):
    """Offsets past 32 bits: rows of a matrix of over 4 GiB whose rows are 2^20
    elements apart."""
    M, D, ld = 2100, 40, 1 << 20
    rng = np.random.default_rng(21)
    x, w = draws(rng, "bf16", M, D), draws(rng, "bf16", D, 24)
    nbytes = M * ld * 2
    p = lib.lib.volta_hip_device_alloc(nbytes)
    if not p:
        pytest.skip("no 4.4 GB of device memory")
    try:
        packed = Mat(lib, "bf16", M, D, x)
        # spread the rows out with the operator itself: y = x, p = 0
        ops.Dropout(M, D, "bf16", 0.0, ld_y=ld).forward(packed, int(p))
        y1, y2 = Mat(lib, "bf16", M, 24), Mat(lib, "bf16", M, 24)
        mw = Mat(lib, "bf16", D, 24, w)
        one, far = ops.Linear(M, D, 24, "bf16"), ops.Linear(M, D, 24, "bf16", ld_x=ld)
        ws = Space(lib, one)
        one.forward(packed, mw, y1, workspace=ws)
        far.forward(int(p), mw, y2, workspace=ws)
        assert np.array_equal(y1.bits(), y2.bits())
        n1, n2 = Mat(lib, "bf16", M, D), Mat(lib, "bf16", M, D)
        ops.RmsNorm(M, D, "bf16", EPS).forward(packed, n1)
        ops.RmsNorm(M, D, "bf16", EPS, ld_x=ld).forward(int(p), n2)
        assert np.array_equal(n1.bits(), n2.bits())
        back = Mat(lib, "bf16", M, D)
        ops.Dropout(M, D, "bf16", 0.0, ld_x=ld).forward(int(p), back)
        assert np.array_equal(back.bits(), packed.bits())
    finally:
        lib.lib.volta_hip_device_free(int(p))


@pytest.mark.parametrize("t", TYPES)
def test_misaligned_beside_an_operand_laid_out_anew(lib, t):
    """x's rows are not whole chunks, so it would be copied; W's are, but W
    starts at an odd element, so neither takes the direct loads: the sums are
    whole numbers, so the result is exact."""
    M, K, N = 1600, 1001, 1504
    rng = np.random.default_rng(78)
    x, w = whole(rng, M, K), whole(rng, K, N)
    op = ops.Linear(M, K, N, t)
    for lead in (0, 1):
        mx, mw, my = Mat(lib, t, M, K, x), Mat(lib, t, K, N, w, lead=lead), Mat(lib, t, M, N)
        ws = Space(lib, op)
        op.forward(mx, mw, my, workspace=ws)
        ws.check()
        assert np.array_equal(my.bits().view(R.STORE[t]), R.pack(x @ w, t)), lead


@pytest.mark.parametrize("t", TYPES)
def test_one_matrix_as_gate_and_up(lib, t):
    """Wg and Wu may be the same matrix, odd rows of it among them."""
    for M, K, N in ((3, 40, 24), (70, 33, 41), (1600, 1001, 1501)):
        rng = np.random.default_rng(M)
        x, w = draws(rng, t, M, K), draws(rng, t, K, N)
        mx, m1, m2 = Mat(lib, t, M, K, x), Mat(lib, t, K, N, w), Mat(lib, t, K, N, w)
        op = ops.GatedFF(M, K, N, t)
        ws, wsb = Space(lib, op), Space(lib, op, True)
        got = []
        for up in (m1, m2):
            h, g, u, dx = Mat(lib, t, M, N), Mat(lib, t, M, N), Mat(lib, t, M, N), Mat(lib, t, M, K)
            op.forward(mx, m1, up, h, gate=g, up=u, workspace=ws)
            op.backward(h, mx, m1, up, g, u, dx=dx, workspace=wsb)
            got.append([m.bits() for m in (h, g, u, dx)])
        ws.check()
        wsb.check()
        assert np.array_equal(got[0][1], got[0][2])
        assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_blocks_on_two_streams_at_once(lib):
    """Two blocks enqueued on two streams, a workspace each, one of them in
    the forms for a few rows: the bits they have alone."""
    hip = _hip(lib)
    blocks = [Block(lib, "bf16", 300, 512, 1024), Block(lib, "bf16", 5, 2048, 4096, seed=12)]
    want = []
    for b in blocks:
        b.run()
        want.append(b.bits())
    streams = [C.c_void_p(), C.c_void_p()]
    for st in streams:
        assert hip.hipStreamCreate(C.byref(st)) == 0
    for _ in range(3):
        for b in blocks:
            for k in Block.OUT:  # spoil the last outputs
                m = b.m[k]
                lib.lib.volta_hip_copy(m.dev.ptr, m.before.ctypes.data, m.before.nbytes, 1)
        assert hip.hipDeviceSynchronize() == 0
        for _ in range(4):
            for b, st in zip(blocks, streams):
                b.run(stream=st.value)
        for st in streams:
            assert hip.hipStreamSynchronize(st) == 0
        for b, w in zip(blocks, want):
            assert all(np.array_equal(v, w[k]) for k, v in b.bits().items())
    for st in streams:
        assert hip.hipStreamDestroy(st) == 0


@pytest.mark.parametrize("t", TYPES)
def test_dropout_at_the_end_of_the_stream(lib, t):
    """Outputs are counted modulo 2^64."""
    M, N, p = 3, 37, 0.5
    rng = np.random.default_rng(4)
    x = draws(rng, t, M, N)
    mx, my = Mat(lib, t, M, N, x), Mat(lib, t, M, N)
    for seed, offset in (((1 << 64) - 1, (1 << 64) - 7), (5, (1 << 64) - 1), (0, 1 << 63)):
        ops.Dropout(M, N, t, p).forward(mx, my, seed=seed, offset=offset)
        want = np.where(R.splitmix_keep(M * N, seed, offset, p).reshape(M, N), 2 * x, 0)
        assert np.array_equal(my.bits().view(R.STORE[t]), R.pack(want, t))


def test_host_memory_refused(lib):
    """A matrix or workspace that is not memory a device reads is refused on
    the host, and nothing is enqueued."""
    M, K, N = 300, 64, 64
    m = {k: Mat(lib, "f32", *s) for k, s in {"x": (M, K), "w": (K, N), "y": (M, N), "dw": (K, N), "r": (1, M)}.items()}
    host = np.zeros(M * N + 4, np.float32)
    h = host.ctypes.data + -host.ctypes.data % 16
    lin, nrm, drp = ops.Linear(M, K, N, act="relu"), ops.RmsNorm(M, K), ops.Dropout(M, K)
    ws = Space(lib, lin, True)

    def refused(name, call):
        with pytest.raises(ops.OperatorError) as e:
            call()
        assert name + " is not memory" in str(e.value), str(e.value)

    refused("x", lambda: lin.forward(h, m["w"], m["y"], workspace=ws))
    refused("w", lambda: lin.forward(m["x"], h, m["y"], workspace=ws))
    refused("y", lambda: lin.forward(m["x"], m["w"], h, workspace=ws))
    refused("bias", lambda: lin.forward(m["x"], m["w"], m["y"], bias=h, workspace=ws))
    refused("dw", lambda: lin.backward(m["y"], m["x"], m["w"], pre=m["y"], dw=h, workspace=ws))
    refused("the workspace", lambda: lin.backward(m["y"], m["x"], m["w"], pre=m["y"], dw=m["dw"], workspace=h))
    refused("weight", lambda: nrm.forward(m["x"], m["y"], weight=h))
    refused("rstd", lambda: nrm.forward(m["x"], m["y"], rstd=h))
    refused("y", lambda: drp.forward(m["x"], h))
    assert all(v.untouched() for v in m.values()) and not host.any()
