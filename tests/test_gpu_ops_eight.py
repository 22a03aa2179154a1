"""e4m3 codes and the linear layer of them (include/volta_ops.h,
volta_amd.ops.Quantize and Linear8) on the GPU: codes and scales bit for bit
against the same arithmetic on the host, products on every tile exactly, the
layer against 64 bits; odd sizes, strides, NaN and infinities, graphs.

Tolerances.  A product of two codes has 8 bits, so a sum of K of them in 32
bits is off by at most K 2^-24 of the sum of the products' magnitudes; the
blocks' sums are scaled (the product of the scales and the fused multiply-add
round once each) and added: 3 + blocks roundings more.  For results of 16 bits
the instruction for codes drops of eight products what is under 2^-17 of the
largest (measured: with one product of 2^16 among them, 2^-1 is lost and 2^0
kept; and its own tests' codes, 128 products of one sign, off by 2^-10.5 of the
largest): 2^-17 of the block's largest for each product."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_graph import Captured, put, spoil
from tests.ops_ref import TYPES, Mat, act, act_error, check, rounded
from tests.test_gpu_ops import Layout, Space, draws, say
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
U = 2.0**-24
TILES = {"256": 0, "256x128": 1, "128": 2, "64x128": 3, "64": 4, "skinny16": 5, "skinny32": 6, "skinny64": 7}
VALUES = R.unpack(np.arange(127, dtype=np.uint8), "e4m3")  # of the codes 0 .. 126


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def encode(v):
    """Floats of up to 448.0001 as codes, to the nearest, ties to even; NaN as 0x7f."""
    a = np.abs(np.asarray(v, np.float64))
    i = np.clip(np.searchsorted(VALUES, a), 1, 126)
    lo, hi = VALUES[i - 1], VALUES[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    code = np.where(np.isnan(a), 0x7F, np.where(up, i, i - 1)).astype(np.uint8)
    return code | np.where(np.signbit(v), 0x80, 0).astype(np.uint8)


def code_matrix(lib, codes, ld=None, lead=0):
    """A matrix of codes as a Mat."""
    m = Mat(lib, "e4m3", *codes.shape, ld=ld, lead=lead)
    host = m.before.copy()
    if codes.size:
        m._view(host)[:, :] = codes
    m.before = host
    assert lib.lib.volta_hip_copy(m.dev.ptr, host.ctypes.data, host.nbytes, 1) == 0
    return m


def groups_of(x, by):
    """Codes and scales of float32 values, in the arithmetic of the header."""
    x = np.asarray(x, np.float32)
    m, c = x.shape
    if by == "blocks":
        x = np.ascontiguousarray(x.T)
        m, c = c, m
        parts = np.pad(x, ((0, -m % 128), (0, -c % 128))).reshape(-(-m // 128), 128, -(-c // 128), 128)
        big = np.abs(parts).max((1, 3))
    else:
        parts = np.pad(x, ((0, 0), (0, -c % 128))).reshape(m, -1, 128)
        big = np.abs(parts).max(2) if m else np.zeros((0, parts.shape[1]), np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        scales = big.astype(np.float32) / np.float32(448)
        scales = np.where(scales < np.float32(2.0**-126), np.float32(2.0**-126), scales).astype(np.float32)
        inv = np.float32(1) / scales
        v = parts * (inv[:, None, :, None] if by == "blocks" else inv[:, :, None])
    v = v.reshape(-1, v.shape[-1] * v.shape[-2] if by != "blocks" else v.shape[2] * 128)[:m, :c]
    return encode(v.astype(np.float32)), scales


SIZES = [(1, 1), (1, 128), (3, 130), (5, 1000), (16, 16), (17, 127), (128, 128), (129, 257), (200, 384), (300, 72)]


@pytest.mark.parametrize("by", ["rows", "blocks"])
@pytest.mark.parametrize("t", TYPES)
def test_codes(lib, t, by):
    for n, (M, N) in enumerate(SIZES):
        for style in ("packed", "odd", "wide"):
            say(t, by, M, N, style)
            rng, L = np.random.default_rng(n), Layout(lib, t, style)
            v = draws(rng, t, M, N) * np.where(rng.random(N) < 0.05, 16.0, 1.0)
            v[:, : N // 3] *= 2.0**-20 if t != "f16" else 2.0**-4
            if M * N > 4000:
                v[:128, :128] = 0
            v = R.unpack(R.pack(v, t), t)
            shape = (N, M) if by == "blocks" else (M, N)
            x, y = L(M, N, v), Mat(lib, "e4m3", *shape, ld=shape[1] + L.pad, lead=L.lead)
            codes, scales = groups_of(v, by)
            s = Mat(lib, "f32", *scales.shape)
            ops.Quantize(M, N, t, by=by, ld_x=x.ld, ld_y=y.ld).forward(x, y, s)
            assert np.array_equal(s.bits().view(np.float32), scales)
            got = y.bits()
            assert np.array_equal(got & 0x7F, codes & 0x7F) and np.array_equal(got[codes & 0x7F != 0], codes[codes & 0x7F != 0])


@pytest.mark.parametrize("t", TYPES)
def test_codes_of_nan_and_infinities(lib, t):
    """NaN: its group's scale and codes; an infinity: an infinite scale, itself NaN, the rest 0."""
    v = np.ones((4, 300))
    v[1, 130], v[2, 5], v[3, 299] = np.nan, np.inf, -np.inf
    x, y, s = Mat(lib, t, 4, 300, v), Mat(lib, "e4m3", 4, 300), Mat(lib, "f32", 4, 3)
    ops.Quantize(4, 300, t).forward(x, y, s)
    got, sc = y.bits(), s.get()
    assert np.isnan(sc[1, 1]) and (got[1, 128:256] & 0x7F == 0x7F).all() and (got[1, :128] == 0x7E).all()
    assert sc[2, 0] == np.inf and got[2, 5] & 0x7F == 0x7F and not (np.delete(got[2, :128], 5) & 0x7F).any()
    assert sc[3, 2] == np.inf and got[3, 299] & 0x7F == 0x7F and (got[3, 128:256] == 0x7E).all()
    y2, s2 = Mat(lib, "e4m3", 300, 4), Mat(lib, "f32", 3, 1)
    ops.Quantize(4, 300, t, by="blocks").forward(x, y2, s2)
    got, sc = y2.bits(), s2.get()[:, 0]
    assert sc[0] == np.inf and np.isnan(sc[1]) and sc[2] == np.inf
    assert (got[128:256] & 0x7F == 0x7F).all() and got[5, 2] & 0x7F == 0x7F and not (got[:5] & 0x7F).any()


def test_codes_as_the_norm_leaves_them(lib):
    """Of the norm's values, where both have them: its output in float32 quantized again."""
    rng = np.random.default_rng(4)
    x = Mat(lib, "f32", 33, 500, draws(rng, "f32", 33, 500))
    y, codes, s = Mat(lib, "f32", 33, 500), [Mat(lib, "e4m3", 33, 500) for _ in range(2)], [Mat(lib, "f32", 33, 4) for _ in range(2)]
    ops.RmsNorm(33, 500).forward(x, y)
    ops.RmsNorm(33, 500, out="e4m3", group=128).forward(x, codes[0], scales=s[0])
    ops.Quantize(33, 500).forward(y, codes[1], s[1])
    assert np.array_equal(codes[0].bits(), codes[1].bits()) and np.array_equal(s[0].bits(), s[1].bits())


SHAPES = [(1, 16, 1), (5, 48, 33), (16, 128, 32), (17, 144, 65), (64, 272, 130), (130, 640, 257), (300, 1040, 520),
          (257, 2048, 136)]


def test_products_on_every_tile(lib):
    """Codes of small whole numbers and scales of powers of two: every sum is exact."""
    whole = encode(np.arange(-8, 9))
    for n, (M, K, N) in enumerate(SHAPES):
        rng = np.random.default_rng(n)
        xc, wc = rng.choice(whole, (M, K)), rng.choice(whole, (N, K))
        blocks = -(-K // 128)
        sx, sw = 2.0 ** rng.integers(-2, 3, (M, blocks)), 2.0 ** rng.integers(-2, 3, (-(-N // 128), blocks))
        xv, wv = R.unpack(xc, "e4m3"), R.unpack(wc, "e4m3")
        for group in (128, 0):
            rows = sx if group else sx[:, :1]
            full = xv * np.repeat(rows, 128 if group else K, 1)[:, :K]
            want = full @ (wv * np.repeat(np.repeat(sw, 128, 0)[:N], 128, 1)[:, :K]).T
            msx, msw = Mat(lib, "f32", *rows.shape, rows), Mat(lib, "f32", *sw.shape, sw)
            for tile, code in TILES.items():
                for direct in (True, False):
                    if not direct and tile in ("256", "256x128", "64x128"):
                        continue
                    for t in TYPES if n % 3 == 0 else ("f32",):
                        for splits in (1, 3):
                            say(M, K, N, "group", group, "tile", tile, "direct", direct, t, "splits", splits)
                            x = code_matrix(lib, xc, ld=K + (16 if direct else 3), lead=0 if direct else 1)
                            w = code_matrix(lib, wc, ld=K + (32 if direct else 5), lead=0 if direct else 3)
                            out = Mat(lib, t, M, N, ld=N + 3, lead=1)
                            rc = lib.lib.volta_hip_op_product8(
                                R.TYPES.index(t), code, splits, int(direct), C.c_void_p(x.ptr), C.c_int64(x.ld),
                                C.c_void_p(msx.ptr), group, C.c_void_p(w.ptr), C.c_int64(w.ld), C.c_void_p(msw.ptr),
                                C.c_void_p(out.ptr), C.c_int64(out.ld), M, N, K)
                            assert rc == 0
                            got = out.bits().view(R.STORE[t])
                            assert np.array_equal(got, R.pack(want, t)), "product"


LAYERS = [(1, 16, 8), (1, 1000, 300), (3, 1, 5), (16, 256, 512), (17, 65, 31), (50, 384, 100), (64, 1024, 64),
          (65, 40, 264), (200, 300, 130), (384, 512, 256), (300, 1000, 700), (0, 24, 16)]
ACTS = ["identity", "relu", "sigmoid", "tanh", "leaky_relu", "silu", "gelu"]


@pytest.mark.parametrize("style", ["packed", "odd", "wide"])
@pytest.mark.parametrize("t", TYPES)
def test_linear8(lib, t, style):
    for n, (M, K, N) in enumerate(LAYERS):
        a, rng, L = ACTS[n % len(ACTS)], np.random.default_rng(n), Layout(lib, t, style)
        bias, residual, group = n % 2 == 0, n % 3 != 1, 0 if n % 4 == 1 else 128
        say(t, style, a, M, K, N, "bias", bias, "residual", residual, "group", group)
        blocks = -(-K // 128)
        xc, wc = rng.integers(0, 256, (M, K)).astype(np.uint8), rng.integers(0, 256, (N, K)).astype(np.uint8)
        xc[xc & 0x7F == 0x7F], wc[wc & 0x7F == 0x7F] = 0, 0
        sx = (np.exp(rng.standard_normal((M, blocks if group else 1))) / 200).astype(np.float32)
        sw = (np.exp(rng.standard_normal((-(-N // 128), blocks))) * K**-0.5 / 100).astype(np.float32)
        b, r = draws(rng, t, N), draws(rng, t, M, N)
        xs = np.repeat(sx.astype(np.float64), 128 if group else K, 1)[:, :K] * R.unpack(xc, "e4m3")
        ws_ = np.repeat(np.repeat(sw.astype(np.float64), 128, 0)[:N], 128, 1)[:, :K] * R.unpack(wc, "e4m3")
        x, w = code_matrix(lib, xc, ld=K + L.pad, lead=L.lead), code_matrix(lib, wc, ld=K + L.pad, lead=L.lead)
        msx, msw = Mat(lib, "f32", M, sx.shape[1], sx), Mat(lib, "f32", *sw.shape, sw)
        y, mr, mb = L(M, N), L(M, N, r), L.vec(N, b)
        op = ops.Linear8(M, K, N, t, a, group=group, ld_x=x.ld, ld_w=w.ld, ld_y=L.ld(N), ld_residual=L.ld(N))
        space = Space(lib, _NoDirection(op))
        op.forward(x, msx, w, msw, y, bias=mb if bias else None, residual=mr if residual else None, workspace=space)
        p = xs @ ws_.T + (b if bias else 0)
        ep = (K + blocks + 4) * U * (np.abs(xs) @ np.abs(ws_).T) + 2 * U * np.abs(p)
        if t != "f32" and M:
            for i in range(0, K, 128):
                ep = ep + 128 * 2.0**-17 * (np.abs(xs[:, None, i:i + 128]) * np.abs(ws_[None, :, i:i + 128])).max(2)
        want = act(a, p)[0] + (r if residual else 0)
        tol = 1.2 * ep + (act_error(t, p)[0] if a not in ("identity", "relu") else 0) + 2 * U * np.abs(want)
        check(y.get(), R.held(want, t), 1.01 * tol + rounded(want, t), "y")
        space.check()
        if residual and M:  # the residual in y's place
            before = y.bits()
            op.forward(x, msx, w, msw, mr, bias=mb if bias else None, residual=mr, workspace=space)
            assert np.array_equal(mr.bits(), before)


class _NoDirection:
    """workspace_bytes as Space asks for it."""

    def __init__(self, op):
        self.op = op

    def workspace_bytes(self, backward=False):
        return self.op.workspace_bytes()


def test_nan_codes_and_scales_stay_in_their_rows(lib):
    """A NaN code reaches its row (x) or column (w) alone, a NaN scale its row or its 128 columns; codes and scales
    behind a matrix's end have no say."""
    M, K, N = 40, 200, 300
    rng = np.random.default_rng(0)
    xc, wc = encode(rng.standard_normal((M, K))), encode(rng.standard_normal((N, K)))
    sx, sw = np.ones((M, 2), np.float32), np.ones((3, 2), np.float32)
    xc[7, 150], wc[201, 3], sx[11, 1], sw[2, 0] = 0x7F, 0xFF, np.nan, np.nan
    want = np.zeros((M, N), bool)
    want[7], want[11], want[:, 201], want[:, 256:] = True, True, True, True
    for pad in (0, 56):  # through copies, and direct from rows with NaN codes behind them
        x, w, y = code_matrix(lib, xc, ld=K + pad), code_matrix(lib, wc, ld=K + pad), Mat(lib, "bf16", M, N)
        op = ops.Linear8(M, K, N, "bf16", ld_x=K + pad, ld_w=K + pad)
        op.forward(x, Mat(lib, "f32", M, 2, sx), w, Mat(lib, "f32", 3, 2, sw), y, workspace=Space(lib, _NoDirection(op)))
        assert np.array_equal(np.isnan(y.get()), want)


def test_a_served_layer_in_a_graph(lib):
    """Norm to codes, product, activation to codes, product onto the residual:
    captured once and replayed on other values, each replay as the eager calls,
    which are near the same layers in 64 bits."""
    M, D, H = 50, 320, 700
    rng = np.random.default_rng(6)
    w1, w2 = draws(rng, "bf16", D, H, scale=D**-0.5), draws(rng, "bf16", H, D, scale=H**-0.5)
    weights = []
    for v in (w1, w2):
        k, n = v.shape
        codes, s = Mat(lib, "e4m3", n, k), Mat(lib, "f32", -(-n // 128), -(-k // 128))
        ops.Quantize(k, n, "bf16", by="blocks").forward(Mat(lib, "bf16", k, n, v), codes, s)
        weights += [codes, s]
    norm, q = ops.RmsNorm(M, D, "bf16", out="e4m3", group=128), ops.Quantize(M, H, "bf16")
    up, down = ops.Linear8(M, D, H, "bf16", "silu"), ops.Linear8(M, H, D, "bf16")

    class Run:
        def __init__(self):
            self.m = {"n": Mat(lib, "e4m3", M, D), "sn": Mat(lib, "f32", M, 3), "h": Mat(lib, "bf16", M, H),
                      "h8": Mat(lib, "e4m3", M, H), "sh": Mat(lib, "f32", M, 6), "y": Mat(lib, "bf16", M, D)}
            self.ws = [Space(lib, _NoDirection(op)) for op in (up, down)]

        def __call__(self, x, stream=0):
            m = self.m
            norm.forward(x, m["n"], scales=m["sn"], stream=stream)
            up.forward(m["n"], m["sn"], weights[0], weights[1], m["h"], workspace=self.ws[0], stream=stream)
            q.forward(m["h"], m["h8"], m["sh"], stream=stream)
            down.forward(m["h8"], m["sh"], weights[2], weights[3], m["y"], residual=x, workspace=self.ws[1], stream=stream)

    x, run, eager = Mat(lib, "bf16", M, D, np.zeros((M, D))), Run(), Run()
    graph = Captured(lib, lambda stream: run(x, stream))
    for i in range(4):
        v = draws(rng, "bf16", M, D, scale=4.0**i)
        put(lib, x, v)
        for m in run.m.values():
            spoil(lib, m)
        eager(x)
        graph.replay()
        for k in run.m:
            assert np.array_equal(run.m[k].bits(), eager.m[k].bits()), k
        n = v / np.sqrt((v**2).mean(1, keepdims=True) + 1e-6)
        h = act("silu", n @ w1)[0]
        want = h @ w2
        # codes are within 2^-4 of their values, at random: four such roundings of every product's factors
        off = np.linalg.norm(run.m["y"].get() - v - want) / np.linalg.norm(want)
        assert off < 4 * 2.0**-4 + np.linalg.norm(v) / np.linalg.norm(want) * 2.0**-8, off
    graph.close()
