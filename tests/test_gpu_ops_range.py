"""The feed-forward operators' gradients (include/volta_ops.h) where their
inputs are far from 1: float16 pre-activation gradients past its largest value
or below its smallest normal one, rows of the norm whose 1/rms has no cube in 32
bits, pre-activations whose square is infinite.  Bounds as in
tests/test_gpu_ops.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import HALF, Mat, act, act_error, check, rounded
from tests.test_gpu_ops import Block, Space, U32, _hip, draws, sum_error
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return load_hip()


SHAPES = [(1, 40, 24), (7, 33, 65), (40, 64, 136), (300, 256, 128), (1100, 1000, 1501)]
# (what dy or dh, up, x and W are multiplied by): past 65504 with results well inside, and where
# float16 has one to five bits left
SCALES = {"large": (30000.0, 40.0, 2.0**-12, 2.0**-12), "small": (2.0**-20, 0.25, 64.0, 64.0)}


def _product_error(p, d, ed, K, want, t):
    """Of p @ d, d off by ed and rounded to t in units in which its largest
    magnitude is at least 2^14: half a step of a subnormal is then 2^-25 2^-14
    of that magnitude."""
    e = ed + HALF[t] * (np.abs(d) + ed) + (np.abs(d) + ed).max() * 2.0**-39
    return 1.001 * (np.abs(p) @ e + sum_error(p, np.abs(d) + e, K) + rounded(want, t)) + 1e-37


@pytest.mark.parametrize("size", SCALES)
@pytest.mark.parametrize("t", R.TYPES)
def test_gated_gradients_far_from_one(lib, t, size):
    """dg = dh u act'(g) is over 65504, or under 2^-14, in most places; dx and
    dW are ordinary numbers of the type."""
    sd, su, sx, sw = SCALES[size]
    for n, (M, K, N) in enumerate(SHAPES):
        a, rng = ("silu", "gelu", "relu")[n % 3], np.random.default_rng(500 + n)
        print(t, size, a, M, K, N, flush=True)
        x, wg, wu = draws(rng, t, M, K, scale=sx), draws(rng, t, K, N, scale=sw), draws(rng, t, K, N, scale=sw)
        dh, g, u = np.clip(draws(rng, t, M, N, scale=sd), -60000, 60000), draws(rng, t, M, N), draws(rng, t, M, N, scale=su)
        dh = R.unpack(R.pack(dh, t), t)
        op = ops.GatedFF(M, K, N, t, a)
        ws = Space(lib, op, True)
        m = [Mat(lib, t, *v.shape, v) for v in (dh, x, wg, wu, g, u)]
        out = {"dx": Mat(lib, t, M, K), "dw_gate": Mat(lib, t, K, N), "dw_up": Mat(lib, t, K, N)}
        op.backward(*m, workspace=ws, **out)
        f, slope = act(a, g)
        ef, es = act_error(t, g) if a != "relu" else (0, 0)
        dg, du = dh * u * slope, dh * f
        eg = np.abs(dh * u) * es + 3 * U32 * np.abs(dg)
        eu = np.abs(dh) * ef + 3 * U32 * np.abs(du)
        cat, ecat, wcat = np.hstack([dg, du]), np.hstack([eg, eu]), np.hstack([wg, wu])
        want = dg @ wg.T + du @ wu.T
        assert np.abs(want).max() < 60000
        check(out["dx"].get(), want, _product_error(wcat, cat.T, ecat.T, 2 * N, want.T, t).T, "dx")
        top = np.abs(cat).max() * 2.0**-39  # both matrices in the same units
        for name, d, ed in (("dw_gate", dg, eg), ("dw_up", du, eu)):
            want = x.T @ d
            assert np.abs(want).max() < 60000
            check(out[name].get(), want, _product_error(x.T, d, ed + top, M, want, t), name)
        ws.check()
        for some in (["dx"], ["dw_gate", "dw_up"]):  # alone, the same bits
            again = {k: Mat(lib, t, out[k].rows, out[k].cols) for k in some}
            op.backward(*m, workspace=ws, **again)
            assert all(np.array_equal(again[k].bits(), out[k].bits()) for k in some)


@pytest.mark.parametrize("size", SCALES)
@pytest.mark.parametrize("t", R.TYPES)
def test_linear_gradients_far_from_one(lib, t, size):
    """dp = dy act'(p): GELU's slope is up to 1.13, so dp passes 65504 where dy
    nearly does."""
    sd, su, sx, sw = SCALES[size]
    for n, (M, K, N) in enumerate(SHAPES):
        rng = np.random.default_rng(550 + n)
        print(t, size, M, K, N, flush=True)
        x, w, p = draws(rng, t, M, K, scale=sx), draws(rng, t, K, N, scale=sw), draws(rng, t, M, N, scale=1.5)
        dy = np.copysign(rng.uniform(60000, 65000, (M, N)), rng.standard_normal((M, N))) if size == "large" else \
            sd * su * rng.standard_normal((M, N))
        dy = R.unpack(R.pack(dy, t), t)
        op = ops.Linear(M, K, N, t, "gelu")
        ws = Space(lib, op, True)
        m = [Mat(lib, t, *v.shape, v) for v in (dy, x, w, p)]
        dx, dw = Mat(lib, t, M, K), Mat(lib, t, K, N)
        op.backward(m[0], m[1], m[2], pre=m[3], dx=dx, dw=dw, workspace=ws)
        slope = act("gelu", p)[1]
        d = dy * slope
        ed = np.abs(dy) * act_error(t, p)[1] + 2 * U32 * np.abs(d)
        want = d @ w.T
        check(dx.get(), want, _product_error(w, d.T, ed.T, N, want.T, t).T, "dx")
        want = x.T @ d
        check(dw.get(), want, _product_error(x.T, d, ed, M, want, t), "dw")
        ws.check()


def test_infinity_keeps_to_its_row_in_dx(lib):
    """A row of dy with an infinity or a NaN spoils its own row of dx alone, and
    rows of zeros stay zeros."""
    M, K, N = 70, 48, 40
    rng = np.random.default_rng(60)
    for bad in (np.inf, np.nan):
        x, w, p, dy = (draws(rng, "f16", *s) for s in ((M, K), (K, N), (M, N), (M, N)))
        dy[5] = 0
        clean = dy.copy()
        dy[3, 7] = bad
        op = ops.Linear(M, K, N, "f16", "silu")
        ws, dx = Space(lib, op, True), Mat(lib, "f16", M, K)
        m = [Mat(lib, "f16", *v.shape, v) for v in (dy, x, w, p)]
        op.backward(m[0], m[1], m[2], pre=m[3], dx=dx, workspace=ws)
        got, d = dx.get(), clean * act("silu", p)[1]
        want = d @ w.T
        tol = _product_error(w, d.T, (np.abs(clean) * act_error("f16", p)[1]).T, N, want.T, "f16").T
        # units of a matrix with an infinity are the type's own: its subnormals end at 2^-25
        tol = tol + np.abs(np.ones((M, N)) @ np.abs(w.T)) * 2.0**-25
        rest = np.arange(M) != 3
        check(got[rest], want[rest], tol[rest], "dx")
        assert not np.isfinite(got[3]).any() and (got[5] == 0).all()


def test_gradients_of_zeros_are_zeros(lib):
    M, K, N = 20, 16, 24
    rng = np.random.default_rng(61)
    op = ops.GatedFF(M, K, N, "f16")
    ws = Space(lib, op, True)
    m = [Mat(lib, "f16", *v.shape, v) for v in (np.zeros((M, N)), draws(rng, "f16", M, K), draws(rng, "f16", K, N),
                                                draws(rng, "f16", K, N), draws(rng, "f16", M, N), draws(rng, "f16", M, N))]
    dx, dg, du = Mat(lib, "f16", M, K), Mat(lib, "f16", K, N), Mat(lib, "f16", K, N)
    op.backward(*m, dx=dx, dw_gate=dg, dw_up=du, workspace=ws)
    assert all((v.get() == 0).all() for v in (dx, dg, du))


# ---------------------------------------------------------------------------
# The norm's gradient.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("eps,scale", [(1e-6, 1e15), (1e-6, 1e16), (0.0, 1e-15), (0.0, 1e-17), (0.0, 1.0)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_norm_gradients_of_rows_far_from_one(lib, t, eps, scale):
    """The cube of rstd, which the formula has, leaves 32 bits from rows of
    1e13 or 1e-13 on; dx and its two terms do not.  Rows held in registers, of
    a wave and of a block, and those read twice."""
    for n, (M, D) in enumerate([(3, 7), (5, 512), (4, 1000), (3, 2056), (2, 9000), (2, 34001)]):
        rng = np.random.default_rng(600 + n)
        print(t, eps, scale, M, D, flush=True)
        dy, s, w = draws(rng, t, M, D, scale=0.1), draws(rng, t, M, D, scale=scale), draws(rng, t, D)
        # the gradient that reaches s by the residual stream, of dx's own size
        ds = draws(rng, t, M, D, scale=0.1 / scale) if n % 2 else None
        rstd32 = (1 / np.sqrt((s**2).mean(1) + eps)).astype(np.float32)
        rstd = rstd32.astype(np.float64)[:, None]
        op = ops.RmsNorm(M, D, t, eps)
        ws = Space(lib, op, True)
        dx, dw = Mat(lib, t, M, D), Mat(lib, t, 1, D)
        op.backward(Mat(lib, t, M, D, dy), Mat(lib, t, M, D, s), Mat(lib, "f32", 1, M, rstd32[None]), dx=dx,
                    weight=Mat(lib, t, 1, D, w), dsum=Mat(lib, t, M, D, ds) if ds is not None else None, dweight=dw,
                    workspace=ws)
        hat, wdy = s * rstd, w * dy
        c = (wdy * hat).mean(1, keepdims=True)
        ec = (D + 6) * U32 * np.abs(wdy * hat).mean(1, keepdims=True)
        want = rstd * (wdy - hat * c) + (ds if ds is not None else 0)
        tol = rstd * (4 * U32 * np.abs(wdy) + np.abs(hat) * (ec + 8 * U32 * np.abs(c))) + 3 * U32 * np.abs(want)
        check(dx.get(), want, 1.01 * tol + rounded(want, t) * 1.01, "dx")
        want = (dy * hat).sum(0)[None]
        tol = (M + 4) * U32 * np.abs(dy * hat).sum(0)[None]
        check(dw.get(), want, 1.01 * tol + rounded(want, t) * 1.01, "dweight")
        ws.check()


# ---------------------------------------------------------------------------
# Slopes of activations.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t", R.TYPES)
def test_gelu_slope_of_large_values(lib, t):
    """1 on the right, 0 on the left, also where x^2 leaves 32 bits; f is x and
    0.  Of one row the biases' gradients are dp, dg and du themselves."""
    big = [40.0, 1000.0, 6e4] + ([1e13, 1e18, 2e19, 1e30, 3e38] if t != "f16" else [])
    x = R.unpack(R.pack([v for b in big for v in (b, -b)], t), t)[None]
    N = x.size
    one, dy = Mat(lib, t, 1, N, np.ones((1, N))), Mat(lib, t, 1, N, np.ones((1, N)))
    pre, inp, w = Mat(lib, t, 1, N, x), Mat(lib, t, 1, 8, np.zeros((1, 8))), Mat(lib, t, 8, N, np.zeros((8, N)))
    lin, gat = ops.Linear(1, 8, N, t, "gelu"), ops.GatedFF(1, 8, N, t, "gelu")
    db, dbg, dbu = Mat(lib, t, 1, N), Mat(lib, t, 1, N), Mat(lib, t, 1, N)
    lin.backward(dy, inp, w, pre=pre, db=db, workspace=Space(lib, lin, True))
    gat.backward(dy, inp, w, w, pre, one, db_gate=dbg, db_up=dbu, workspace=Space(lib, gat, True))
    assert np.array_equal(db.get(), (x > 0) * 1.0) and np.array_equal(dbg.get(), (x > 0) * 1.0)
    assert np.array_equal(dbu.get(), np.where(x > 0, x, 0.0))


@pytest.mark.parametrize("t", R.TYPES)
def test_gelu_slope_of_nan_is_nan(lib, t):
    N = 8
    pre = Mat(lib, t, 1, N, np.where(np.arange(N) == 3, np.nan, 1.0)[None])
    m = [Mat(lib, t, 1, N, np.ones((1, N))) for _ in range(2)]
    w, db = Mat(lib, t, N, N, np.zeros((N, N))), Mat(lib, t, 1, N)
    lin = ops.Linear(1, N, N, t, "gelu")
    lin.backward(m[0], m[1], w, pre=pre, db=db, workspace=Space(lib, lin, True))
    assert np.array_equal(np.isnan(db.get()[0]), np.arange(N) == 3)


# ---------------------------------------------------------------------------
# Float16 gradients' units, which live in the workspace, in a captured graph.
# ---------------------------------------------------------------------------
def test_float16_block_in_a_graph_with_other_inputs(lib):
    """The block in float16, captured once and replayed on other values of dy,
    eager runs of another block between the replays: each replay finds its own
    units."""
    hip = _hip(lib)
    b, other = Block(lib, "f16", 70, 96, 200), Block(lib, "f16", 33, 64, 96, seed=12)
    scales = (1.0, 2.0**-9, 64.0, 2.0**-14, 1.0)
    dys = [R.unpack(R.pack(b.v["dy"] * s, "f16"), "f16") for s in scales]

    def put(dy):
        m = b.m["dy"]
        host = m.before.copy()
        m._view(host)[:, :] = R.pack(dy, "f16").view(R.BITS["f16"])
        m.before = host
        assert lib.lib.volta_hip_copy(m.dev.ptr, host.ctypes.data, host.nbytes, 1) == 0

    want = []
    for dy in dys:
        put(dy)
        b.run()
        want.append(b.bits())
    st, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreate(C.byref(st)) == 0
    assert hip.hipStreamBeginCapture(st, 1) == 0  # thread-local
    b.run(stream=st.value)
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
    for dy, w in zip(dys, want):
        put(dy)
        other.run()
        assert hip.hipDeviceSynchronize() == 0
        assert hip.hipGraphLaunch(run, st) == 0
        assert hip.hipStreamSynchronize(st) == 0
        assert all(np.array_equal(v, w[k]) for k, v in b.bits().items())
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    assert hip.hipStreamDestroy(st) == 0
