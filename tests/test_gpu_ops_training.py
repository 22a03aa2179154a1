"""The operators as a program uses them together: a block and an output layer
trained (norm, gated layer, linear layer onto the residual, norm, loss over the
classes; gradients of all of them; the weights updated by orthogonalised
momentum), and the trained block served from e4m3 codes."""
from __future__ import annotations

import numpy as np
import pytest

from tests.ops_graph import Captured, put
from tests.ops_ref import HALF, TYPES, Mat, act, check
from tests.test_gpu_ops import Space, draws
from tests.test_gpu_ops_eight import _NoDirection
from tests.test_gpu_ops_loss import Words
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def lib():
    return load_hip()


class Model:
    """s = x; h = silu(n Wg) * (n Wu), n = norm(s); y = s + h Wd; loss of
    norm(y) Wo + bo.  `step` runs it forward, back, and updates Wg, Wu, Wd and
    Wo."""

    def __init__(self, lib, t, M, D, H, C, seed=1, lr=0.02):
        self.lib, self.t, self.dims, self.lr = lib, t, (M, D, H, C), lr
        rng = np.random.default_rng(seed)
        self.v = {"wn1": 1 + draws(rng, t, D, scale=0.1), "wn2": 1 + draws(rng, t, D, scale=0.1),
                  "wgu": draws(rng, t, 2 * D, H, scale=D**-0.5), "wd": draws(rng, t, H, D, scale=H**-0.5),
                  "wo": draws(rng, t, D, C, scale=D**-0.5), "bo": draws(rng, t, C, scale=0.1)}
        self.m = {k: self._mat(v) for k, v in self.v.items()}
        for k, s in {"x": (M, D), "n1": (M, D), "g": (M, H), "u": (M, H), "h": (M, H), "y": (M, D), "n2": (M, D),
                     "dn2": (M, D), "dy": (M, D), "dh": (M, H), "dn1": (M, D), "dx": (M, D), "dwn1": (1, D),
                     "dwn2": (1, D), "dwgu": (2 * D, H), "dwd": (H, D), "dwo": (D, C), "dbo": (1, C)}.items():
            self.m[k] = Mat(lib, t, *s, np.zeros(s))
        for k, s in {"r1": (1, M), "r2": (1, M), "loss": (1, M), "lse": (1, M), "dloss": (1, M)}.items():
            self.m[k] = Mat(lib, "f32", *s, np.full(s, 1.0 / M))
        for k in ("wgu", "wd", "wo"):
            self.m["m_" + k] = Mat(lib, "f32", *self.v[k].shape, np.zeros(self.v[k].shape))
        self.labels = Words(lib, np.zeros(M))
        self.norm, self.gated = ops.RmsNorm(M, D, t, EPS), ops.GatedFF(M, D, H, t)
        self.down, self.loss = ops.Linear(M, H, D, t), ops.CrossEntropy(M, D, C, t)
        # the two matrices of the gated layer are one batch
        self.update = {"wgu": ops.Muon(D, H, t, batch=2), "wd": ops.Muon(H, D, t), "wo": ops.Muon(D, C, t)}
        spaces = [Space(lib, o, b) for o in (self.norm, self.gated, self.down, self.loss) for b in (False, True)]
        spaces += [Space(lib, _NoDirection(o)) for o in self.update.values()]
        self.ws = max(spaces, key=lambda s: s.nbytes)

    def _mat(self, v):
        return Mat(self.lib, self.t, *(v.shape if v.ndim == 2 else (1, v.size)), v)

    def half(self, k):
        """The second matrix of a pair."""
        return self.m[k].ptr + self.dims[1] * self.dims[2] * (4 if self.t == "f32" else 2)

    def forward(self, stream=0):
        m, kw = self.m, {"workspace": self.ws, "stream": stream}
        self.norm.forward(m["x"], m["n1"], weight=m["wn1"], rstd=m["r1"], stream=stream)
        self.gated.forward(m["n1"], m["wgu"], self.half("wgu"), m["h"], gate=m["g"], up=m["u"], **kw)
        self.down.forward(m["h"], m["wd"], m["y"], residual=m["x"], **kw)
        self.norm.forward(m["y"], m["n2"], weight=m["wn2"], rstd=m["r2"], stream=stream)
        self.loss.forward(m["n2"], m["wo"], self.labels, m["loss"], lse=m["lse"], bias=m["bo"], **kw)

    def backward(self, stream=0):
        m, kw = self.m, {"workspace": self.ws, "stream": stream}
        self.loss.backward(m["n2"], m["wo"], self.labels, m["lse"], m["dloss"], bias=m["bo"], dx=m["dn2"], dw=m["dwo"],
                           db=m["dbo"], **kw)
        self.norm.backward(m["dn2"], m["y"], m["r2"], m["dy"], weight=m["wn2"], dweight=m["dwn2"], **kw)
        self.down.backward(m["dy"], m["h"], m["wd"], dx=m["dh"], dw=m["dwd"], **kw)
        self.gated.backward(m["dh"], m["n1"], m["wgu"], self.half("wgu"), m["g"], m["u"], dx=m["dn1"], dw_gate=m["dwgu"],
                            dw_up=self.half("dwgu"), **kw)
        self.norm.backward(m["dn1"], m["x"], m["r1"], m["dx"], weight=m["wn1"], dsum=m["dy"], dweight=m["dwn1"], **kw)

    def step(self, stream=0):
        self.forward(stream)
        self.backward(stream)
        for k, op in self.update.items():
            op.step(self.m[k], self.m["d" + k], self.m["m_" + k], self.lr, decay=0.01, workspace=self.ws, stream=stream)

    def forward64(self, x, labels, **other):
        v, D = {**self.v, **other}, self.dims[1]
        n1 = x / np.sqrt((x**2).mean(1, keepdims=True) + EPS) * v["wn1"]
        y = x + act("silu", n1 @ v["wgu"][:D])[0] * (n1 @ v["wgu"][D:]) @ v["wd"]
        z = y / np.sqrt((y**2).mean(1, keepdims=True) + EPS) * v["wn2"] @ v["wo"] + v["bo"]
        top = z.max(1, keepdims=True)
        loss = top[:, 0] + np.log(np.exp(z - top).sum(1)) - z[np.arange(len(z)), np.maximum(labels, 0)]
        return np.where(labels < 0, 0.0, loss), y


def test_gradients_against_differences(lib):
    """In float32: the derivative of the mean loss along a direction of every
    weight, against central differences of the model in 64 bits (their error is
    1e-10 of the third derivative; the chain's sums are within 1e-5 of their
    magnitudes)."""
    M, D, H, C = 40, 24, 36, 50
    b = Model(lib, "f32", M, D, H, C)
    rng = np.random.default_rng(3)
    x, labels = draws(rng, "f32", M, D), rng.integers(-1, C, M)
    put(lib, b.m["x"], x)
    b.labels = Words(lib, labels)
    b.forward()
    b.backward()
    want, _ = b.forward64(x, labels)
    check(b.m["loss"].get()[0], want, 2e-5 * (1 + np.abs(want)), "loss")
    for k in ("wn1", "wn2", "wgu", "wd", "wo", "bo", "x"):
        v = rng.standard_normal((b.v[k] if k != "x" else x).shape)
        eps = 1e-5
        if k == "x":
            up, dn = (b.forward64(x + e * v, labels)[0].sum() for e in (eps, -eps))
        else:
            up, dn = (b.forward64(x, labels, **{k: b.v[k] + e * v})[0].sum() for e in (eps, -eps))
        slope, g = (up - dn) / (2 * eps) / M, b.m["d" + k].get().reshape(v.shape)
        assert abs((g * v).sum() - slope) <= 2e-5 * (np.abs(g) * np.abs(v)).sum() + 1e-7, k


@pytest.mark.parametrize("t", TYPES)
def test_steps_in_a_graph(lib, t):
    """Whole training steps, captured once: three replays, on other data each,
    leave the weights and momenta that three eager steps do, bit for bit, and
    weights that are numbers."""
    dims = (96, 64, 160, 300)
    a, b, other = Model(lib, t, *dims), Model(lib, t, *dims), Model(lib, t, 33, 40, 56, 70, seed=2)
    graph = Captured(lib, a.step)
    rng = np.random.default_rng(4)
    for _ in range(3):
        x, labels = draws(rng, t, dims[0], dims[1]), rng.integers(-1, dims[3], dims[0]).astype(np.int32)
        for m in (a, b):
            put(lib, m.m["x"], x)
            assert lib.lib.volta_hip_copy(m.labels.ptr, labels.ctypes.data, labels.nbytes, 1) == 0
        b.step()
        other.step()
        graph.replay()
        for k in ("wgu", "wd", "wo", "m_wgu", "m_wd", "m_wo", "loss", "dx", "dwn1", "dbo"):
            assert np.array_equal(a.m[k].bits(), b.m[k].bits()), k
            assert np.isfinite(a.m[k].get()).all(), k
    assert not np.array_equal(a.m["wd"].get(), a.v["wd"])
    graph.close()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_the_trained_block_served_from_codes(lib, t):
    """Two steps of training, then the block from e4m3 codes of its weights and
    activations: near its 16-bit form.  A code is within 2^-4 of its value and,
    at random, some 0.4 of that (a uniform error over a step of 2^-3 to 2^-4);
    a product of two such rounded operands is off by sqrt(2) times that of its
    norm, and the second product's operand by the first one's."""
    M, D, H, C = 130, 192, 400, 60
    b = Model(lib, t, M, D, H, C)
    rng = np.random.default_rng(5)
    x = draws(rng, t, M, D)
    put(lib, b.m["x"], x)
    b.labels = Words(lib, rng.integers(0, C, M))
    b.step()
    b.step()
    b.forward()
    want, h16 = b.m["y"].get() - x, b.m["h"].get()
    codes = {}
    for k, at, rows, cols in (("g", b.m["wgu"].ptr, D, H), ("u", b.half("wgu"), D, H), ("d", b.m["wd"].ptr, H, D)):
        c, s = Mat(lib, "e4m3", cols, rows), Mat(lib, "f32", -(-cols // 128), -(-rows // 128))
        ops.Quantize(rows, cols, t, by="blocks").forward(at, c, s)
        codes[k] = (c, s)
    n, sn = Mat(lib, "e4m3", M, D), Mat(lib, "f32", M, 2)
    ops.RmsNorm(M, D, t, EPS, out="e4m3", group=128).forward(b.m["x"], n, weight=b.m["wn1"], scales=sn)
    g, u, y = Mat(lib, t, M, H), Mat(lib, t, M, H), Mat(lib, t, M, D)
    for name, out, a in (("g", g, "silu"), ("u", u, "identity")):
        op = ops.Linear8(M, D, H, t, a)
        op.forward(n, sn, *codes[name], out, workspace=Space(lib, _NoDirection(op)))
    h = g.get() * u.get()
    one = 0.4 * 2.0**-4
    assert np.linalg.norm(h - h16) / np.linalg.norm(h16) < 2 * np.sqrt(2) * np.sqrt(2) * one  # two products, each of two
    mh, h8, sh = Mat(lib, t, M, H, h), Mat(lib, "e4m3", M, H), Mat(lib, "f32", M, 4)
    ops.Quantize(M, H, t).forward(mh, h8, sh)
    op = ops.Linear8(M, H, D, t)
    op.forward(h8, sh, *codes["d"], y, residual=b.m["x"], workspace=Space(lib, _NoDirection(op)))
    got = y.get() - x
    tol = 2 * np.sqrt(6) * one * np.linalg.norm(want) + 2 * HALF[t] * np.linalg.norm(x)
    assert np.linalg.norm(got - want) < tol, (np.linalg.norm(got - want), tol)
