"""The update by orthogonalised momentum (include/volta_ops.h,
volta_amd.ops.Muon) on the GPU: its products on every tile exactly, the result
against 64 bits, momentum and weights, batches, odd sizes and strides, zeros,
NaN, far values, graphs.

Tolerances.  The iteration amplifies errors of X's small singular directions,
by what follows from the matrix, so the bound comes from the matrix: the same
iteration with X, G and the polynomials rounded as the kernels round them is off
by some distance, and the kernels, whose roundings are others of the same sizes,
by up to three times it.  bfloat16: to float16 in units of a power of two over
the range, but for the diagonals of G and the polynomials, which are kept at
sides of up to 256 and of one to more than four; the sums' 32 bits are nothing beside that.  float16 and float32: to two such numbers
(23 bits), and a sum of K products is a chain of K / 8 additions, each
rounded to 24 bits (the instruction adds eight products at a time: 99 % of its
results over random operands are those of that chain; with the smaller two of
the three products first, those of the rests add nothing to it); the product of the two rests, which is left out, is
2^-24 of the others; and alpha d + beta r is rounded to 24 bits three times,
which together is as much as the two numbers' half step (the first form of this
bound had left it out).  The result's rounding adds half a step.  The coefficients
are floats in the call, and so in the reference."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_graph import Captured, put, spoil
from tests.ops_ref import HALF, TYPES, Mat
from tests.test_gpu_ops import Layout, draws, say, whole
from tests.test_gpu_ops_eight import _NoDirection
from tests.test_gpu_ops import Space as _Space
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
ABC = tuple(float(np.float32(v)) for v in (3.4445, -4.7750, 2.0315))


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def space(lib, op):
    return _Space(lib, _NoDirection(op))


def mixed(alpha, d, beta, r):
    """alpha d + beta r in float32."""
    d, r = (np.float32(k) * v.astype(np.float32) for k, v in ((alpha, d), (beta, r)))
    return (d + r).astype(np.float64)


def iterate(u, steps=5, coefficients=ABC, eps=1e-7, rounding=lambda v, kind: v, mul=lambda p, q: p @ q,
            mix=lambda alpha, d, beta, r: alpha * d + beta * r):
    a, b, c = coefficients
    x = u / (np.sqrt((u**2).sum()) + eps) if u.any() else u
    x = rounding(x, 1.0)
    tall = x.shape[0] > x.shape[1]
    for i in range(steps):
        g = rounding(mul(x.T, x) if tall else mul(x, x.T), -1.5)  # < 0: a diagonal may be kept
        p = rounding(mix(c, mul(g, g), b, g), -4.0)
        x = mix(1.0, mul(x, p) if tall else mul(p, x), a, x)
        if i < steps - 1:
            x = rounding(x, 1.25)
    return x


def halves(v, bound):
    """To float16 in the unit that holds |bound|; bound < 0: but for the diagonal."""
    unit = 2.0 ** (15 - np.ceil(np.log2(abs(bound))))
    got = (v * unit).astype(np.float16).astype(np.float64) / unit
    if bound < 0:
        np.fill_diagonal(got, np.diag(v))
    return got


def pairs(v, bound):
    """To two float16 numbers in that unit."""
    unit = 2.0 ** (15 - np.ceil(np.log2(abs(bound))))
    first = (v * unit).astype(np.float16).astype(np.float64)
    return (first + (v * unit - first).astype(np.float16).astype(np.float64)) / unit


def chain(p, q):
    """p q, eight products added to the sum at a time, the sum rounded to float32."""
    d = np.zeros((p.shape[0], q.shape[1]), np.float32)
    for k in range(0, p.shape[1], 8):
        d = (d + p[:, k:k + 8] @ q[k:k + 8]).astype(np.float32)
    return d.astype(np.float64)


def before_rounding(t, u, want, **kw):
    """The 2-norm by which the X of a result of type t may be off."""
    small, large = sorted((-n % 8 + n for n in u.shape))
    kept = small <= 256 or large > 4 * small  # the diagonals
    half = lambda v, bound: halves(v, bound if kept else abs(bound))  # noqa: E731
    near = iterate(u, rounding=half, **kw) if t == "bf16" else iterate(u, rounding=pairs, mul=chain, mix=mixed, **kw)
    return 3 * np.linalg.norm(near - want)


def allowed(t, u, want, **kw):
    """The 2-norm by which a result of type t may be off."""
    return before_rounding(t, u, want, **kw) + (HALF[t] + 2.0**-22) * np.linalg.norm(want) + R.FLOOR[t] * np.sqrt(want.size)


def planes(lib, v, n):
    """Matrices of whole numbers as float16, or as two planes of it."""
    rows = v.reshape(-1, v.shape[-1])
    first = rows.astype(np.float16).astype(np.float64)
    return Mat(lib, "f16", n * rows.shape[0], rows.shape[1], rows if n == 1 else np.concatenate([first, rows - first]))


def _blend(lib, n, layout, kind, tile, splits, batch, p, q, r, out, M, N, K):
    return lib.lib.volta_hip_op_blend(n, layout, kind, tile, splits, batch, C.c_void_p(p.ptr), C.c_void_p(q.ptr),
                                      C.c_void_p(r.ptr), C.c_void_p(out.ptr), M, N, K, C.c_float(0.5), C.c_float(-2.0))


def both(out, n):
    v = out.get()
    return v if n == 1 else v[:len(v) // 2] + v[len(v) // 2:]


@pytest.mark.parametrize("n", [1, 2])
def test_products_on_every_tile(lib, n):
    """Whole numbers, with two planes some of 12 bits: alpha P Q + beta r is
    exact, whatever the tile, the layout and the splits."""
    for k, (batch, M, N, K) in enumerate([(1, 8, 8, 8), (3, 16, 72, 40), (2, 136, 64, 264), (5, 8, 200, 8), (1, 264, 520, 136),
                                          (2, 304, 128, 72)]):
        rng = np.random.default_rng(k)
        P, Q, r = whole(rng, batch, M, K), whole(rng, batch, K, N), whole(rng, batch, M, N)
        if n == 2:  # a row of P and columns of Q with a second number, none of which meet
            P[:, 1, :] += 2049
            Q[:, :, 2] = 0
            Q[:, K // 2, 2] = 4097  # one: |0.5 3 4097 + 2 5001| stays in float16's range, a sum of them would not
            P[:, 1, :] *= rng.random(K) < 0.02
            r[:, 3, 5] = 5001
        want = 0.5 * (P @ Q) - 2 * r
        if n == 2:
            want[:, 1, 2] = 0  # both have rests there
        mp, mr = planes(lib, P, n), planes(lib, r, n)
        for layout in (0, 1):
            mq = planes(lib, np.ascontiguousarray(Q.swapaxes(1, 2)) if layout == 1 else Q, n)
            for tile in range(5):
                for splits in (1, 3):
                    say("planes", n, "batch", batch, M, N, K, "layout", layout, "tile", tile, "splits", splits)
                    out = Mat(lib, "f16", n * batch * M, N)
                    assert _blend(lib, n, layout, 6, tile, splits, batch, mp, mq, mr, out, M, N, K) == 0
                    got = both(out, n).reshape(want.shape).copy()
                    if n == 2:
                        got[:, 1, 2] = 0
                    assert np.array_equal(got, want)


@pytest.mark.parametrize("n", [1, 2])
def test_symmetric_products_on_every_tile(lib, n):
    """Of X X^T: half of the tiles computed, all stored, exactly."""
    for k, (batch, M, K) in enumerate([(1, 8, 8), (3, 72, 40), (2, 136, 264), (5, 8, 200), (1, 520, 136), (2, 304, 72),
                                       (1, 1096, 24)]):
        rng = np.random.default_rng(k)
        X, r = whole(rng, batch, M, K), whole(rng, batch, M, M)
        r = r + r.swapaxes(1, 2)
        if n == 2:
            r += 4097
        want = 0.5 * (X @ X.swapaxes(1, 2)) - 2 * r
        mr = planes(lib, r, n)
        for layout in (1, 2):
            mx = planes(lib, X if layout == 1 else np.ascontiguousarray(X.swapaxes(1, 2)), n)
            for tile in (0, 2, 4):
                for splits in (1, 3):
                    say("planes", n, "batch", batch, M, K, "layout", layout, "tile", tile, "splits", splits)
                    out = Mat(lib, "f16", n * batch * M, M)
                    assert _blend(lib, n, layout, 7, tile, splits, batch, mx, mx, mr, out, M, M, K) == 0
                    assert np.array_equal(both(out, n).reshape(want.shape), want)


SIZES = [(1, 1, 1), (3, 1, 9), (2, 9, 1), (1, 16, 16), (4, 17, 33), (2, 64, 50), (1, 100, 300), (3, 130, 70), (1, 256, 256),
         (1, 40, 1000), (2, 1000, 24), (1, 300, 301), (5, 8, 8), (3, 96, 97), (2, 105, 128), (1, 128, 2000), (2, 136, 129), (1, 30, 576)]


def gradients(rng, batch, m, n):
    """A few strong directions and noise, as a layer's gradient has."""
    return rng.standard_normal((batch, m, n)) + 0.5 * rng.standard_normal((batch, m, 4)) @ rng.standard_normal((batch, 4, n))


@pytest.mark.parametrize("style", ["packed", "odd", "wide"])
@pytest.mark.parametrize("t", TYPES)
def test_orthogonalize(lib, t, style):
    for k, (batch, m, n) in enumerate(SIZES):
        rng, L = np.random.default_rng(k), Layout(lib, t, style)
        say(t, style, batch, m, n)
        v = R.unpack(R.pack(gradients(rng, batch, m, n), t), t)
        u, o = L(batch * m, n, v.reshape(-1, n)), L(batch * m, n)
        op = ops.Muon(m, n, t, batch=batch, ld_u=L.ld(n), ld_o=L.ld(n))
        ws = space(lib, op)
        op.orthogonalize(u, o, workspace=ws)
        got = o.get().reshape(batch, m, n)
        for z in range(batch):
            want = iterate(v[z])
            off = np.linalg.norm(got[z] - want)
            assert off <= allowed(t, v[z], want), (z, off, allowed(t, v[z], want))
        ws.check()
        before = o.bits()
        op.orthogonalize(u, u, workspace=ws)  # in place
        assert np.array_equal(u.bits(), before)


@pytest.mark.parametrize("t", TYPES)
def test_larger(lib, t):
    """Sizes whose products take the larger tiles and split sums."""
    # the last two take two steps at once, wide and tall
    for k, (batch, m, n) in enumerate([(1, 512, 2000), (2, 1100, 520), (1, 72, 9000), (1, 5000, 96), (16, 384, 1500),
                                       (20, 1400, 330), (1, 136, 9000), (1, 7000, 200), (1, 384, 2880)]):
        rng = np.random.default_rng(50 + k)
        say(t, batch, m, n)
        v = R.unpack(R.pack(gradients(rng, batch, m, n), t), t)
        u, o = Mat(lib, t, batch * m, n, v.reshape(-1, n)), Mat(lib, t, batch * m, n)
        op = ops.Muon(m, n, t, batch=batch)
        ws = space(lib, op)
        op.orthogonalize(u, o, workspace=ws)
        got = o.get().reshape(batch, m, n)
        for z in range(batch):
            if z % 9 == 0 or batch < 16:
                want = iterate(v[z])
                assert np.linalg.norm(got[z] - want) <= allowed(t, v[z], want), z
        ws.check()


@pytest.mark.parametrize("t", TYPES)
def test_scaled_permutations(lib, t):
    """Equal singular values: the result is the permutation times what the
    polynomial makes of one value, and exactly 0 elsewhere; whatever the scale,
    from where squares leave 32 bits."""
    rng = np.random.default_rng(1)
    n = 72
    for power in ((0, 60, -60, 120) if t != "f16" else (0, 10, -10)):
        perm = np.eye(n)[rng.permutation(n)] * 2.0**power
        u, o = Mat(lib, t, n, n, perm), Mat(lib, t, n, n)
        op = ops.Muon(n, n, t, eps=0.0)
        op.orthogonalize(u, o, workspace=space(lib, op))
        s = 1 / np.sqrt(n)
        for _ in range(5):
            s = ABC[0] * s + ABC[1] * s**3 + ABC[2] * s**5
        got = o.get()
        assert not got[perm == 0].any()
        # five steps' roundings of X, G and B, amplified by slopes of at most 3.45 (s is under 1.21): 3.45^5 of each
        assert np.abs(got[perm != 0] / s - 1).max() <= 500 * (2.0**-12 if t == "bf16" else 2.0**-24) + HALF[t]


@pytest.mark.parametrize("t", TYPES)
def test_steps_and_coefficients(lib, t):
    rng = np.random.default_rng(8)
    v = R.unpack(R.pack(gradients(rng, 1, 40, 60), t), t)
    u = Mat(lib, t, 40, 60, v[0])
    for steps, abc, eps in ((1, ABC, 1e-7), (2, ABC, 0.5), (12, (1.875, -1.25, 0.375), 1e-7), (3, (1.5, -0.5, 0.0), 0.0),
                            (1, (1.0, 0.0, 0.0), 0.0)):
        op = ops.Muon(40, 60, t, steps=steps, coefficients=abc, eps=eps)
        o = Mat(lib, t, 40, 60)
        op.orthogonalize(u, o, workspace=space(lib, op))
        kw = {"steps": steps, "coefficients": tuple(float(np.float32(c)) for c in abc), "eps": eps}
        want = iterate(v[0], **kw)
        assert np.linalg.norm(o.get() - want) <= allowed(t, v[0], want, **kw), (steps, abc)


@pytest.mark.parametrize("t", TYPES)
def test_zeros_and_nan_stay_in_their_matrix(lib, t):
    rng = np.random.default_rng(2)
    v = R.unpack(R.pack(gradients(rng, 5, 33, 20), t), t)
    v[1], v[2, 3, 4], v[4, 0, 0] = 0, np.nan, np.inf
    for eps in (1e-7, 0.0):
        op, o = ops.Muon(33, 20, t, batch=5, eps=eps), Mat(lib, t, 5 * 33, 20)
        op.orthogonalize(Mat(lib, t, 5 * 33, 20, v.reshape(-1, 20)), o, workspace=space(lib, op))
        got = o.get().reshape(5, 33, 20)
        assert not got[1].any() and np.isnan(got[2]).all() and np.isnan(got[4]).all()
        for z in (0, 3):
            want = iterate(v[z], eps=eps)
            assert np.linalg.norm(got[z] - want) <= allowed(t, v[z], want, eps=eps)


@pytest.mark.parametrize("style", ["packed", "odd"])
@pytest.mark.parametrize("t", TYPES)
def test_step(lib, t, style):
    """Momentum in the arithmetic of 32 bits, weights from its orthogonal matrix, in place and apart."""
    for k, (batch, m, n, nesterov) in enumerate([(1, 64, 200, True), (3, 50, 17, False), (2, 1, 30, True), (1, 300, 100, True)]):
        rng, L = np.random.default_rng(k), Layout(lib, t, style)
        say(t, style, batch, m, n, nesterov)
        lr, beta, decay, scale = 0.05, 0.9, 0.2, 1.5
        g = R.unpack(R.pack(gradients(rng, batch, m, n), t), t)
        mom = rng.standard_normal((batch, m, n)).astype(np.float32)
        w = draws(rng, t, batch, m, n, scale=0.1)
        b32 = np.float32(beta)
        m32 = b32 * mom + g.astype(np.float32)
        u = (g.astype(np.float32) + b32 * m32 if nesterov else m32).astype(np.float64)
        mg, mw, w_out = L(batch * m, n, g.reshape(-1, n)), L(batch * m, n, w.reshape(-1, n)), L(batch * m, n)
        L32 = Layout(lib, "f32", style)
        mm, m_out = L32(batch * m, n, mom.reshape(-1, n)), L32(batch * m, n)
        op = ops.Muon(m, n, t, batch=batch, ld_u=L.ld(n), ld_m=L.ld(n), ld_o=L.ld(n))
        ws = space(lib, op)
        kw = dict(beta=beta, nesterov=nesterov, decay=decay, scale=scale, workspace=ws)
        op.step(mw, mg, mm, lr, w_out=w_out, momentum_out=m_out, **kw)
        assert np.array_equal(m_out.bits().view(np.float32).reshape(m32.shape), m32)
        assert np.array_equal(mm.bits().view(np.float32).reshape(mom.shape), mom)
        got = w_out.get().reshape(w.shape)
        step = float(np.float32(lr) * np.float32(scale))
        keep = float(np.float32(1) - np.float32(lr) * np.float32(decay))
        for z in range(batch):
            x = iterate(u[z])
            want = keep * w[z] - step * x
            tol = step * before_rounding(t, u[z], x) + (HALF[t] + 2.0**-22) * np.linalg.norm(np.abs(want) + np.abs(w[z]))
            assert np.linalg.norm(got[z] - want) <= tol, z
        op.step(mw, mg, mm, lr, **kw)  # in place
        assert np.array_equal(mw.bits(), w_out.bits()) and np.array_equal(mm.bits(), m_out.bits())
        ws.check()


@pytest.mark.parametrize("t", TYPES)
def test_in_a_graph(lib, t):
    """Steps captured once and replayed, on other gradients each time: weights
    and momentum follow the eager steps bit for bit."""
    batch, m, n = 2, 96, 160
    rng = np.random.default_rng(3)
    w0, mom0 = draws(rng, t, batch * m, n), np.zeros((batch * m, n))
    op, other = ops.Muon(m, n, t, batch=batch), ops.Muon(40, 30, t)

    class State:
        def __init__(self):
            self.w, self.m, self.ws = Mat(lib, t, batch * m, n, w0), Mat(lib, "f32", batch * m, n, mom0), space(lib, op)

        def step(self, stream=0):
            op.step(self.w, g, self.m, 0.1, decay=0.01, workspace=self.ws, stream=stream)

    g = Mat(lib, t, batch * m, n, np.zeros((batch * m, n)))
    a, b = State(), State()
    ou, oo, ows = Mat(lib, t, 40, 30, draws(rng, t, 40, 30)), Mat(lib, t, 40, 30), space(lib, other)
    graph = Captured(lib, a.step)
    for i in range(4):
        put(lib, g, gradients(rng, batch, m, n).reshape(-1, n) * 10.0 ** (-i))
        b.step()
        other.orthogonalize(ou, oo, workspace=ows)
        graph.replay()
        assert np.array_equal(a.w.bits(), b.w.bits()) and np.array_equal(a.m.bits(), b.m.bits())
        assert np.isfinite(a.w.get()).all()
        spoil(lib, oo)
    graph.close()
