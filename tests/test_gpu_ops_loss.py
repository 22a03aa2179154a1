"""The loss of an output layer (include/volta_ops.h, volta_amd.ops.CrossEntropy)
on the GPU against its definition in 64 bits: every form of its products, odd
sizes, strides, rows without a label, classes taken out, infinities, more
classes than one piece holds, graphs and streams.

Tolerances.  With u = 2^-24: a sum of K products is off by at most (K + 2) u of
the sum of the products' magnitudes, and z by that and 2 u |z| for the bias.
An exponential is off by its argument's error, by |argument| 2^-22 (its
rounding and the factor log2 e's, in units of the result) and by 2^-21 (the
hardware's exp2, or expf).  A sum of positive terms is off by the longest chain
of additions times u.  lse adds the roundings of the logarithm and of the sum
with the largest z, 2 u each.  dz is rounded to the type (half a step); of up to
128 rows it is held as two numbers of the type (half a step of half a step)."""
from __future__ import annotations

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_graph import Captured, put, spoil
from tests.ops_ref import HALF, TYPES, Mat, check, rounded
from tests.test_gpu_ops import Layout, Space, draws, say, sum_error
from volta_amd import DeviceArray, load_hip, ops

pytestmark = pytest.mark.gpu
U = 2.0**-24


@pytest.fixture(scope="module")
def lib():
    return load_hip()


class Words:
    """Class labels in device memory."""

    def __init__(self, lib, v):
        self.dev = DeviceArray(np.asarray(v, np.int32) if len(v) else np.zeros(1, np.int32), lib)
        self.ptr = self.dev.ptr


def reference(x, w, b, labels):
    """z, lse and loss of finite z, in 64 bits; the errors that 32 bits allow them."""
    K, C = w.shape
    z = x @ w + (0 if b is None else b)
    ez = sum_error(x, w, K) + 2 * U * np.abs(z)
    top = z.max(1, keepdims=True)
    ex = np.exp(z - top)
    s = ex.sum(1, keepdims=True)
    p, lse = ex / s, (top + np.log(s))[:, 0]
    e_lse = (p * (ez + np.abs(z - top) * 2.0**-22 + 2.0**-21)).sum(1) + (60 + C / 1024) * U
    e_lse = e_lse + 4 * U * (np.abs(lse) + np.abs(np.log(s[:, 0])))
    has = labels >= 0
    at = np.where(has, labels, 0)
    rows = np.arange(len(labels))
    loss = np.where(has, lse - z[rows, at], 0.0)
    e_loss = np.where(has, e_lse + ez[rows, at] + U * np.abs(loss), 0.0)
    return z, ez, lse, 1.1 * e_lse + 1e-30, loss, 1.1 * e_loss + 1e-30


def gradients(t, x, w, z, ez, lse, labels, dloss, pieces=1, rows=0):
    """dx, dw, db in 64 bits and their tolerances; lse is the float that the call
    takes, `rows` what the call has where x is a few of them."""
    has = labels >= 0
    g = np.where(has, dloss, 0.0)[:, None]
    p = np.exp(z - lse[:, None])
    hit = np.zeros_like(z)
    hit[np.arange(len(labels))[has], labels[has]] = 1
    dz = (p - hit) * g
    floor = 0.0
    if t == "f16" and has.any() and np.abs(g).max() > 0:  # in units: the largest dloss is in [2^14, 2^15)
        floor = 2.0**-25 * np.abs(g).max() * 2.0**-14
    arg = np.abs(z - lse[:, None])
    edz = (p * (ez + 3 * U * (np.abs(lse[:, None]) + np.abs(z)) + arg * 2.0**-22 + 2.0**-21) + 3 * U * np.abs(p - hit))
    C, (M, K) = w.shape[1], x.shape
    twice = t != "f32" and max(M, rows) <= 128
    half, terms = (HALF[t] ** 2, 2 * M) if twice else (HALF[t], M)  # terms of dw: rows of dz
    edz = 1.1 * edz * np.abs(g) + half * np.abs(dz) * 1.01 + np.where(g != 0, floor, 0)
    dx, dw, db = dz @ w.T, x.T @ dz, dz.sum(0)
    tx = 1.01 * (edz @ np.abs(w).T + (C + 5 + 2 * pieces) * U * ((np.abs(dz) + edz) @ np.abs(w).T)) + 1.01 * rounded(dx, t)
    tw = 1.01 * (np.abs(x).T @ edz + (terms + 4) * U * (np.abs(x).T @ (np.abs(dz) + edz))) + 1.01 * rounded(dw, t)
    tb = 1.01 * (edz.sum(0) + (terms + 4) * U * (np.abs(dz) + edz).sum(0)) + 1.01 * rounded(db, t)
    return (dx, tx), (dw, tw), (db, tb)


SIZES = [(1, 8, 16), (1, 1000, 300), (2, 3, 1), (5, 64, 1000), (16, 256, 517), (17, 65, 31), (50, 384, 2), (64, 1024, 96),
         (65, 40, 264), (200, 300, 130), (384, 64, 512), (1, 4096, 10007), (0, 24, 16)]


@pytest.mark.parametrize("style", ["packed", "odd", "wide"])
@pytest.mark.parametrize("t", TYPES)
def test_forward_and_backward(lib, t, style):
    for n, (M, K, C) in enumerate(SIZES):
        rng, L = np.random.default_rng(n), Layout(lib, t, style)
        with_bias = n % 2 == 0
        say(t, style, M, K, C, "bias", with_bias)
        x, w, b = draws(rng, t, M, K), draws(rng, t, K, C, scale=2 * K**-0.5), draws(rng, t, C)
        labels = rng.integers(0, C, M)
        labels[rng.random(M) < 0.2] = -1 - n
        dloss = rng.standard_normal(M).astype(np.float32).astype(np.float64) / max(1, M)
        mx, mw, mb = L(M, K, x), L(K, C, w), L.vec(C, b) if with_bias else None
        ml, loss, lse = Words(lib, labels), Mat(lib, "f32", 1, max(M, 1)), Mat(lib, "f32", 1, max(M, 1))
        op = ops.CrossEntropy(M, K, C, t, ld_x=L.ld(K), ld_w=L.ld(C), ld_dx=L.ld(K), ld_dw=L.ld(C))
        ws = Space(lib, op)
        op.forward(mx, mw, ml, loss, lse=lse, bias=mb, workspace=ws)
        dx, dw, db = L(M, K), L(K, C), L.vec(C)
        wb = Space(lib, op, True)
        if M == 0:
            assert loss.untouched() and lse.untouched()
            op.backward(mx, mw, ml, lse, loss, bias=mb, dx=dx, dw=dw, db=db, workspace=wb)
            assert dx.untouched() and not dw.get().any() and not db.get().any()
            continue
        z, ez, want_lse, e_lse, want, e_loss = reference(x, w, b if with_bias else None, labels)
        check(lse.get()[0], want_lse, e_lse, "lse")
        check(loss.get()[0], want, e_loss, "loss")
        ws.check()
        kept = want_lse.astype(np.float32)
        ml32, md = Mat(lib, "f32", 1, M, kept), Mat(lib, "f32", 1, M, dloss)
        op.backward(mx, mw, ml, ml32, md, bias=mb, dx=dx, dw=dw, db=db, workspace=wb)
        grads = gradients(t, x, w, z, ez, kept.astype(np.float64), labels, dloss)
        for m, name, (v, tol) in zip((dx, dw, db), ("dx", "dw", "db"), grads):
            check(m.get().reshape(v.shape), v, tol, name)
        wb.check()
        # each gradient alone is the same
        for name, m in (("dx", L(M, K)), ("dw", L(K, C)), ("db", L.vec(C))):
            op.backward(mx, mw, ml, ml32, md, bias=mb, **{name: m}, workspace=wb)
            assert np.array_equal(m.bits(), {"dx": dx, "dw": dw, "db": db}[name].bits()), name


TILED = [(300, 512, 520), (1000, 128, 1003), (2048, 64, 2056), (600, 72, 12000), (96, 4096, 128), (33, 8192, 64)]


@pytest.mark.parametrize("t", TYPES)
def test_larger_tiles(lib, t):
    """Sizes whose products take the larger tiles, and sums split over blocks."""
    for n, (M, K, C) in enumerate(TILED):
        rng = np.random.default_rng(100 + n)
        say(t, M, K, C)
        x, w, b = draws(rng, t, M, K), draws(rng, t, K, C, scale=2 * K**-0.5), draws(rng, t, C)
        labels = rng.integers(0, C, M)
        labels[::7] = -1
        dloss = rng.standard_normal(M).astype(np.float32).astype(np.float64) / M
        mx, mw, mb, ml = Mat(lib, t, M, K, x), Mat(lib, t, K, C, w), Mat(lib, t, 1, C, b), Words(lib, labels)
        loss, lse = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)
        op = ops.CrossEntropy(M, K, C, t)
        ws, wb = Space(lib, op), Space(lib, op, True)
        op.forward(mx, mw, ml, loss, lse=lse, bias=mb, workspace=ws)
        z, ez, want_lse, e_lse, want, e_loss = reference(x, w, b, labels)
        check(lse.get()[0], want_lse, e_lse, "lse")
        check(loss.get()[0], want, e_loss, "loss")
        kept = want_lse.astype(np.float32)
        dx, dw, db = Mat(lib, t, M, K), Mat(lib, t, K, C), Mat(lib, t, 1, C)
        op.backward(mx, mw, ml, Mat(lib, "f32", 1, M, kept), Mat(lib, "f32", 1, M, dloss), bias=mb, dx=dx, dw=dw, db=db,
                    workspace=wb)
        for m, name, (v, tol) in zip((dx, dw, db), ("dx", "dw", "db"),
                                     gradients(t, x, w, z, ez, kept.astype(np.float64), labels, dloss)):
            check(m.get().reshape(v.shape), v, tol, name)
        ws.check()
        wb.check()


@pytest.mark.parametrize("t,few", [(t, False) for t in TYPES] + [("bf16", True), ("f16", True)])
def test_classes_in_several_pieces(lib, t, few):
    """More dz than a piece holds: dx is the sum over the pieces, dw's columns
    are each piece's own.  Against the gradients of a few rows and columns in
    64 bits."""
    # few rows: dz is held as two numbers
    M, K, C = (128, 24, 600011) if few else (2048, 24, 70001) if t == "f32" else (4096, 24, 66003)
    rng = np.random.default_rng(7)
    x, w, b = draws(rng, t, M, K), draws(rng, t, K, C, scale=0.3), draws(rng, t, C)
    labels = rng.integers(0, C, M)
    labels[:4] = [0, C - 1, 32768, -1]
    dloss = rng.standard_normal(M).astype(np.float32).astype(np.float64) / M
    op = ops.CrossEntropy(M, K, C, t)
    # two pieces at least, and less than all of dz
    assert M * C * (4 if few or t == "f32" else 2) > 1 << 28
    mx, mw, mb, ml = Mat(lib, t, M, K, x), Mat(lib, t, K, C, w), Mat(lib, t, 1, C, b), Words(lib, labels)
    loss, lse = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)
    ws, wb = Space(lib, op), Space(lib, op, True)
    op.forward(mx, mw, ml, loss, lse=lse, bias=mb, workspace=ws)
    kept = lse.bits().view(np.float32)[0].astype(np.float64)
    dx, dw, db = Mat(lib, t, M, K), Mat(lib, t, K, C), Mat(lib, t, 1, C)
    op.backward(mx, mw, ml, lse, Mat(lib, "f32", 1, M, dloss), bias=mb, dx=dx, dw=dw, db=db, workspace=wb)
    some = np.r_[0:8, M // 2:M // 2 + 8, M - 8:M]
    z, ez, want_lse, e_lse, want, e_loss = reference(x[some], w, b, labels[some])
    check(kept[some], want_lse, e_lse, "lse")
    check(loss.get()[0][some], want, e_loss, "loss")
    top = np.abs(np.where(labels >= 0, dloss, 0)).max()
    (v, tol), _, _ = gradients(t, x[some], w, z, ez, kept[some], labels[some], dloss[some], pieces=3, rows=M)
    if t == "f16":  # units are of the largest dloss of all rows
        tol = tol + 2.0**-25 * top * 2.0**-14 * np.abs(w).sum(1)
    check(dx.get()[some], v, tol, "dx")
    cols = np.r_[0:8, 32760:32776, 65500:65560, C // 2 - 200:C // 2 + 200, C - 5:C]
    zc = x @ w[:, cols] + b[cols]
    ezc = sum_error(x, w[:, cols], K) + 2 * U * np.abs(zc)
    inside = np.full(C, -1)
    inside[cols] = np.arange(len(cols))
    lab = np.where(labels >= 0, inside[labels], -1)
    # rows whose label lies elsewhere still have a gradient: their label hits none of these columns
    wide = np.concatenate([zc, np.full((M, 1), -1e30)], 1)
    lab = np.where(labels < 0, -1, np.where(lab < 0, len(cols), lab))
    _, (v, tol), (vb, tb) = gradients(t, x, np.concatenate([w[:, cols], np.zeros((K, 1))], 1), wide,
                                      np.concatenate([ezc, np.zeros((M, 1))], 1), kept, lab, dloss)
    check(dw.get()[:, cols], v[:, :-1], tol[:, :-1], "dw")
    check(db.get()[0][cols], vb[:-1], tb[:-1], "db")
    ws.check()
    wb.check()


@pytest.mark.parametrize("t", TYPES)
def test_classes_taken_out_and_bad_rows(lib, t):
    """A bias of -inf takes a class out, a whole wave's columns of them too;
    +inf, NaN and rows with no class left give NaN in their row alone; a label
    behind the classes gives NaN, a negative one nothing whatever its row holds."""
    M, K, C = 40, 16, 700
    rng = np.random.default_rng(3)
    x, w = draws(rng, t, M, K), draws(rng, t, K, C, scale=0.5)
    b = np.zeros(C)
    out = np.zeros(C, bool)
    out[128:400] = out[690:] = out[0] = True
    b[out] = -np.inf
    labels = rng.choice(np.flatnonzero(~out), M)
    labels[3] = -5
    labels[4] = 200  # a class that is out: its loss is infinite
    mw, mb = Mat(lib, t, K, C, w), Mat(lib, t, 1, C, b)
    bad = x.copy()
    bad[10, 0] = np.nan
    bad[11, 0] = np.inf
    bad[3, 1] = np.nan  # the row without a label
    mx, ml = Mat(lib, t, M, K, bad), Words(lib, np.r_[labels[:20], C, labels[21:]])
    loss, lse, op = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M), ops.CrossEntropy(M, K, C, t)
    ws, wb = Space(lib, op), Space(lib, op, True)
    op.forward(mx, mw, ml, loss, lse=lse, bias=mb, workspace=ws)
    good = np.array([i for i in range(M) if i not in (3, 4, 10, 11, 20)])
    z, ez, want_lse, e_lse, want, e_loss = reference(x[good], w[:, ~out], None, np.searchsorted(np.flatnonzero(~out), labels[good]))
    got, got_lse = loss.get()[0], lse.get()[0]
    check(got[good], want, e_loss, "loss")
    check(got_lse[good], want_lse, e_lse, "lse")
    assert got[3] == 0 and got[4] == np.inf and np.isfinite(got_lse[4])
    assert np.isnan(got[[10, 11, 20]]).all() and np.isnan(got_lse[[3, 10, 11]]).all() and np.isfinite(got_lse[20])
    # gradients: bad rows in dx alone where their dloss is 0 ... 0 times NaN is NaN: they are given no label
    lab = labels.copy()
    lab[[10, 11, 20]] = -1
    dl = Mat(lib, "f32", 1, M, np.r_[np.full(3, 0.5), np.nan, np.full(M - 4, 0.5)])
    kept = np.where(np.isin(np.arange(M), good), got_lse, np.nan)
    kept[4] = got_lse[4]
    dx, dw, db = Mat(lib, t, M, K), Mat(lib, t, K, C), Mat(lib, t, 1, C)
    zero = x.copy()
    zero[[3, 10, 11, 20]] = 0
    op.backward(Mat(lib, t, M, K, zero), mw, Words(lib, lab), Mat(lib, "f32", 1, M, kept), dl, bias=mb, dx=dx, dw=dw,
                db=db, workspace=wb)
    assert not dx.get()[[3, 10, 11, 20]].any() and np.isfinite(dx.get()).all()
    grad = dw.get()
    assert np.isfinite(grad).all() and not grad[:, out & (np.arange(C) != 200)].any()
    assert db.get()[0][200] == -0.5 and grad[:, 200].any()
    # a label behind the classes: its row, and what it reaches
    lab[20] = C
    op.backward(Mat(lib, t, M, K, zero), mw, Words(lib, lab), Mat(lib, "f32", 1, M, np.where(np.isnan(kept), 1.0, kept)), dl,
                bias=mb, dx=dx, dw=dw, db=db, workspace=wb)
    assert np.isnan(dx.get()[20]).all() and np.isfinite(np.delete(dx.get(), 20, 0)).all() and np.isnan(db.get()).all()
    # no class left
    none = Mat(lib, t, 1, C, np.full(C, -np.inf))
    op.forward(Mat(lib, t, M, K, x), mw, ml, loss, lse=lse, bias=none, workspace=ws)
    assert (lse.get()[0] == -np.inf).all() and np.isnan(loss.get()[0][labels >= 0][:5]).all()


@pytest.mark.parametrize("t", TYPES)
def test_rows_without_labels_alone(lib, t):
    M, K, C = 70, 64, 129
    rng = np.random.default_rng(5)
    mx, mw = Mat(lib, t, M, K, draws(rng, t, M, K)), Mat(lib, t, K, C, draws(rng, t, K, C))
    ml, loss, lse = Words(lib, np.full(M, -1)), Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)
    op = ops.CrossEntropy(M, K, C, t)
    ws, wb = Space(lib, op), Space(lib, op, True)
    op.forward(mx, mw, ml, loss, lse=lse, workspace=ws)
    assert not loss.get().any() and np.isfinite(lse.get()).all()
    alone = Mat(lib, "f32", 1, M)
    op.forward(mx, mw, None, None, lse=alone, workspace=ws)
    assert np.array_equal(alone.bits(), lse.bits())
    dx, dw, db = Mat(lib, t, M, K), Mat(lib, t, K, C), Mat(lib, t, 1, C)
    op.backward(mx, mw, ml, lse, Mat(lib, "f32", 1, M, np.full(M, np.inf)), dx=dx, dw=dw, db=db, workspace=wb)
    assert not dx.get().any() and not dw.get().any() and not db.get().any()


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6])
def test_float16_gradients_of_far_dloss(lib, scale):
    """dz in units: its products keep float16's bits where the results are in its range."""
    M, K, C = 32, 48, 80
    rng = np.random.default_rng(11)
    x, w = draws(rng, "f16", M, K, scale=2.0**-9 if scale > 1 else 1), draws(rng, "f16", K, C, scale=2.0**-9 if scale > 1 else 1)
    labels, dloss = rng.integers(0, C, M), (scale * rng.standard_normal(M)).astype(np.float32).astype(np.float64)
    z, ez, want, _, _, _ = reference(x, w, None, labels)
    kept = want.astype(np.float32)
    op = ops.CrossEntropy(M, K, C, "f16")
    wb, dx, dw = Space(lib, op, True), Mat(lib, "f16", M, K), Mat(lib, "f16", K, C)
    op.backward(Mat(lib, "f16", M, K, x), Mat(lib, "f16", K, C, w), Words(lib, labels), Mat(lib, "f32", 1, M, kept),
                Mat(lib, "f32", 1, M, dloss), dx=dx, dw=dw, workspace=wb)
    grads = gradients("f16", x, w, z, ez, kept.astype(np.float64), labels, dloss)
    for m, (v, tol) in zip((dx, dw), grads):
        check(m.get(), R.held(v, "f16"), tol, "gradient")


def test_gradients_against_differences(lib):
    """The loss' own differences, in float32."""
    M, K, C = 6, 10, 40
    rng = np.random.default_rng(2)
    x, w, b = rng.standard_normal((M, K)), rng.standard_normal((K, C)), rng.standard_normal(C)
    labels = rng.integers(0, C, M)
    labels[2] = -1
    op = ops.CrossEntropy(M, K, C, "f32")
    ws, wb, ml = Space(lib, op), Space(lib, op, True), Words(lib, labels)
    lse, loss = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)

    def total(x, w, b):
        op.forward(Mat(lib, "f32", M, K, x), Mat(lib, "f32", K, C, w), ml, loss, lse=lse, bias=Mat(lib, "f32", 1, C, b),
                   workspace=ws)
        return loss.get().sum()

    total(x, w, b)
    dx, dw, db = Mat(lib, "f32", M, K), Mat(lib, "f32", K, C), Mat(lib, "f32", 1, C)
    op.backward(Mat(lib, "f32", M, K, x), Mat(lib, "f32", K, C, w), ml, lse, Mat(lib, "f32", 1, M, np.ones(M)),
                bias=Mat(lib, "f32", 1, C, b), dx=dx, dw=dw, db=db, workspace=wb)
    for i, g in enumerate((dx.get(), dw.get(), db.get()[0])):
        v = rng.standard_normal(g.shape)
        h = 1e-2
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = args[0][i] + h * v, args[1][i] - h * v
        slope = (total(*args[0]) - total(*args[1])) / (2 * h)
        # a third derivative's h^2 / 6 of at most |v|_1^3-like terms, and 32 bits' noise over h
        assert abs(slope - (g * v).sum()) < 2e-2 * max(1, np.abs(g * v).sum()), i


@pytest.mark.parametrize("t", TYPES)
def test_in_a_graph_with_other_inputs(lib, t):
    """Captured once and replayed on other values, eager calls of another
    problem between the replays: each replay as the eager call."""
    M, K, C = 130, 96, 1003
    op, other = ops.CrossEntropy(M, K, C, t), ops.CrossEntropy(33, 64, 200, t)
    rng = np.random.default_rng(1)

    def problem(M, K, C):
        m = {"x": Mat(lib, t, M, K, np.zeros((M, K))), "w": Mat(lib, t, K, C, np.zeros((K, C))),
             "b": Mat(lib, t, 1, C, np.zeros(C)), "l": Words(lib, rng.integers(-1, C, M)),
             "d": Mat(lib, "f32", 1, M, np.zeros(M))}
        out = [Mat(lib, *s) for s in (("f32", 1, M), ("f32", 1, M), (t, M, K), (t, K, C), (t, 1, C))]
        return m, out

    def run(op, m, out, ws, stream=0):
        loss, lse, dx, dw, db = out
        op.forward(m["x"], m["w"], m["l"], loss, lse=lse, bias=m["b"], workspace=ws, stream=stream)
        op.backward(m["x"], m["w"], m["l"], lse, m["d"], bias=m["b"], dx=dx, dw=dw, db=db, workspace=ws, stream=stream)

    def space(op):
        return max((Space(lib, op), Space(lib, op, True)), key=lambda s: s.nbytes)

    m, out = problem(M, K, C)
    _, eager = problem(M, K, C)
    m2, out2 = problem(33, 64, 200)
    ws, ws_eager, ws2 = space(op), space(op), space(other)
    graph = Captured(lib, lambda stream: run(op, m, out, ws, stream))
    for i in range(5):
        for k in "xwb":
            put(lib, m[k], draws(rng, t, m[k].rows, m[k].cols))
        put(lib, m["d"], rng.standard_normal(M) * 10.0 ** (2 * i - 4))
        for o in out:
            spoil(lib, o)
        run(op, m, eager, ws_eager)
        run(other, m2, out2, ws2)
        graph.replay()
        for a, e in zip(out, eager):
            # no NaN; float16 gradients of the last turn may be past its range: |dloss| of 3e4 times |w| of 3
            assert np.array_equal(a.bits(), e.bits()) and not np.isnan(a.get()).any()
    graph.close()
