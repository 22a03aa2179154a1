"""The loss and the products of codes at sizes whose plans take the tiles that the
other tests' small ones do not, on the GPU: the layer of codes on 256x256 with its
own epilogue and the rows' scales turned, and the statistics and gradients of the
loss on 64x128 and the larger tiles.

Tolerances.  Codes of whole numbers up to 8 with scales of powers of two: blocks of
128 sums of at most 64, times at most 2, 35 of them, in halves of a half: under 2^20 and
exact in 32 bits, in any order; so are biases and residuals of whole numbers.  The
instruction for codes keeps what is not under 2^-17 of the largest of eight products,
all of these.  The loss as in test_gpu_ops_loss.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import ops_ref as R
from tests.ops_ref import TYPES, Mat, act, act_error, check, rounded
from tests.test_gpu_ops import Space, draws, say
from tests.test_gpu_ops_eight import _NoDirection, code_matrix, encode
from tests.test_gpu_ops_loss import Words, gradients, reference
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
WHOLE = encode(np.arange(-8, 9))


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def planned(lib, e, layout, kind, M, N, K):
    """The tile and the splits of a product of aligned operands."""
    got = (C.c_int32 * 3)()
    lib.lib.volta_hip_op_plan(e, layout, kind, C.c_int64(M), C.c_int64(N), C.c_int64(K), 1, 1, 1, got)
    return got[0], got[1]


class Codes:
    """A product of codes whose result is exact."""

    def __init__(self, lib, M, K, N, group, lead=0):
        rng = np.random.default_rng(M + K + N)
        blocks = -(-K // 128)
        xc, wc = rng.choice(WHOLE, (M, K)), rng.choice(WHOLE, (N, K))
        sx = 2.0 ** rng.integers(-1, 1, (M, blocks if group else 1))
        sw = 2.0 ** rng.integers(-1, 2, (-(-N // 128), blocks))
        x = R.unpack(xc, "e4m3") * np.repeat(sx, 128 if group else K, 1)[:, :K]
        w = R.unpack(wc, "e4m3") * np.repeat(np.repeat(sw, 128, 0)[:N], 128, 1)[:, :K]
        self.p = x @ w.T
        assert np.abs(self.p).max() < 60000
        self.x, self.w = code_matrix(lib, xc, lead=lead), code_matrix(lib, wc, lead=lead)
        self.sx, self.sw = Mat(lib, "f32", *sx.shape, sx), Mat(lib, "f32", *sw.shape, sw)
        self.bias = rng.integers(-9, 10, N).astype(float)
        self.residual = rng.integers(-9, 10, (M, N)).astype(float)


@pytest.mark.parametrize("inputs", [4352, 4368])
@pytest.mark.parametrize("group,lead", [(128, 0), (128, 1), (0, 0)])
def test_a_long_prompt_of_codes(lib, inputs, group, lead):
    """Rows and outputs that end inside a tile, a turn of 32 scales and a lane's 8 columns;
    more than 32 blocks of inputs, the last one whole or not (in which case, as for float32
    results, 256x128 runs what is planned as 256x256); through registers from misaligned codes."""
    M, N = 3001, 3003
    c = Codes(lib, M, inputs, N, group, lead)
    assert planned(lib, 1, 1, 0, M, N, inputs)[0] == 0
    for t in TYPES:
        for a, bias, residual in (("identity", True, True), ("relu", False, True), ("silu", True, False)):
            if a == "silu" and (t == "f32" or lead):
                continue
            say(M, inputs, N, "group", group, "lead", lead, t, a)
            op = ops.Linear8(M, inputs, N, t, a, group=group, ld_y=N + 5, ld_residual=N + 5)
            ws = Space(lib, _NoDirection(op))
            # the scales' turn has its own space
            assert (ws.nbytes >= 4 * M * -(-inputs // 128)) == (group == 128)
            y, mb = Mat(lib, t, M, N, ld=N + 5, lead=1), Mat(lib, t, 1, N, c.bias)
            mr = Mat(lib, t, M, N, c.residual, ld=N + 5, lead=1)
            p = c.p + (c.bias if bias else 0)
            want = act(a, p)[0] + (c.residual if residual else 0)
            op.forward(c.x, c.sx, c.w, c.sw, y, bias=mb if bias else None, residual=mr if residual else None, workspace=ws)
            got = y.bits()
            if a == "silu":
                check(y.get(), R.held(want, t), 1.01 * (act_error(t, p)[0] + rounded(want, t)), "y")
            else:
                assert np.array_equal(got.view(R.STORE[t]), R.pack(want, t))
            if residual:  # in y's place
                op.forward(c.x, c.sx, c.w, c.sw, mr, bias=mb if bias else None, residual=mr, workspace=ws)
                assert np.array_equal(mr.bits(), got)
            ws.check()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_the_large_product_of_codes(lib, t):
    """256x256 of 16-bit results at small sizes around its edges, whole and split."""
    for n, (M, K, N) in enumerate([(1, 128, 1), (16, 128, 32), (130, 640, 257), (257, 2048, 136), (600, 384, 300),
                                   (256, 256, 512), (255, 1152, 513)]):
        for group in (128, 0):
            c = Codes(lib, M, K, N, group)
            for splits in (1, 2, 3):
                say(t, M, K, N, "group", group, "splits", splits)
                out = Mat(lib, t, M, N, ld=N + 3, lead=1)
                assert lib.lib.volta_hip_op_product8(
                    R.TYPES.index(t), 0, splits, 1, C.c_void_p(c.x.ptr), C.c_int64(c.x.ld), C.c_void_p(c.sx.ptr), group,
                    C.c_void_p(c.w.ptr), C.c_int64(c.w.ld), C.c_void_p(c.sw.ptr), C.c_void_p(out.ptr), C.c_int64(out.ld),
                    M, N, K) == 0
                assert np.array_equal(out.bits().view(R.STORE[t]), R.pack(c.p, t))


# tile (256, 256x128, 128, 64x128: 0 to 3), split: rows, inputs, classes
LOSSES = {2: [(3, False, 1, 64, 16392), (3, False, 32, 128, 16392), (3, False, 65, 64, 8200), (3, True, 1000, 4096, 264),
              (2, False, 65, 64, 16392), (1, False, 130, 64, 16392), (0, False, 65, 64, 32776)],
          4: [(3, False, 1, 64, 24584), (3, False, 65, 64, 8200), (3, True, 1000, 1024, 264), (2, False, 65, 64, 16392),
              (2, True, 1000, 2048, 264), (1, False, 1000, 64, 4104), (0, False, 1000, 64, 8200)]}


@pytest.mark.parametrize("n", range(7))
@pytest.mark.parametrize("t", TYPES)
def test_losses_on_the_larger_tiles(lib, t, n):
    tile, split, M, K, classes = LOSSES[4 if t == "f32" else 2][n]
    for kind in (3, 4):  # the statistics and dz
        got = planned(lib, 4 if t == "f32" else 2, 0, kind, M, classes, K)
        assert got[0] == tile and (got[1] > 1) == split, got
    rng = np.random.default_rng(n)
    say(t, M, K, classes)
    x, w, b = draws(rng, t, M, K), draws(rng, t, K, classes, scale=2 * K**-0.5), draws(rng, t, classes)
    labels = rng.integers(0, classes, M)
    labels[::7] = -1
    labels[0] = classes - 1
    dloss = rng.standard_normal(M).astype(np.float32).astype(np.float64) / M
    mx, mw, mb, ml = Mat(lib, t, M, K, x), Mat(lib, t, K, classes, w), Mat(lib, t, 1, classes, b), Words(lib, labels)
    loss, lse = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)
    op = ops.CrossEntropy(M, K, classes, t)
    ws, wb = Space(lib, op), Space(lib, op, True)
    op.forward(mx, mw, ml, loss, lse=lse, bias=mb, workspace=ws)
    z, ez, want_lse, e_lse, want, e_loss = reference(x, w, b, labels)
    check(lse.get()[0], want_lse, e_lse, "lse")
    check(loss.get()[0], want, e_loss, "loss")
    kept = want_lse.astype(np.float32)
    dx, dw, db = Mat(lib, t, M, K), Mat(lib, t, K, classes), Mat(lib, t, 1, classes)
    op.backward(mx, mw, ml, Mat(lib, "f32", 1, M, kept), Mat(lib, "f32", 1, M, dloss), bias=mb, dx=dx, dw=dw, db=db,
                workspace=wb)
    for m, name, (v, tol) in zip((dx, dw, db), ("dx", "dw", "db"),
                                 gradients(t, x, w, z, ez, kept.astype(np.float64), labels, dloss)):
        check(m.get().reshape(v.shape), v, tol, name)
    ws.check()
    wb.check()
