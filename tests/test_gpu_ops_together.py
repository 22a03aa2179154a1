"""The operators around the feed-forward layers where calls meet: two programs
on two streams at once, rows far into a large matrix, addresses that are not
16-byte aligned beside ones that are."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests.ops_graph import hip, put, spoil
from tests.ops_ref import TYPES, Mat
from tests.test_gpu_ops import Space, draws, say
from tests.test_gpu_ops_eight import _NoDirection, code_matrix, encode
from tests.test_gpu_ops_loss import Words
from tests.test_gpu_ops_training import Model
from volta_amd import load_hip, ops

pytestmark = pytest.mark.gpu
OUT = ("loss", "lse", "dx", "dwgu", "dwd", "dwo", "dbo")


@pytest.fixture(scope="module")
def lib():
    return load_hip()


def test_two_trainings_on_two_streams_at_once(lib):
    """A workspace each: the weights that either training has alone."""
    h, rng = hip(lib), np.random.default_rng(1)
    dims = [("bf16", (300, 256, 512, 1000)), ("f32", (40, 96, 130, 333))]
    data = [(draws(rng, t, d[0], d[1]), Words(lib, rng.integers(-1, d[3], d[0]))) for t, d in dims]

    def models():
        both = [Model(lib, t, *d) for t, d in dims]
        for m, (x, labels) in zip(both, data):
            put(lib, m.m["x"], x)
            m.labels = labels
        return both

    alone = models()
    for m in alone:
        for _ in range(4):
            m.step()
    both = models()
    streams = [C.c_void_p(), C.c_void_p()]
    for st in streams:
        assert h.hipStreamCreate(C.byref(st)) == 0
    assert h.hipDeviceSynchronize() == 0
    for _ in range(4):
        for m, st in zip(both, streams):
            m.step(stream=st.value)
    for st in streams:
        assert h.hipStreamSynchronize(st) == 0 and h.hipStreamDestroy(st) == 0
    for m, want in zip(both, alone):
        for k in OUT + ("wgu", "wd", "wo", "m_wgu", "m_wd", "m_wo"):
            assert np.array_equal(m.m[k].bits(), want.m[k].bits()), k


def test_rows_far_into_a_large_matrix(lib):
    """Offsets past 32 bits: rows 2^20 elements apart, over 4 GiB of them."""
    M, D, N, ld = 2100, 48, 40, 1 << 20
    rng = np.random.default_rng(21)
    p = lib.lib.volta_hip_device_alloc(M * ld * 2)
    if not p:
        pytest.skip("no 4.4 GB of device memory")
    p = int(p)
    try:
        x, w = Mat(lib, "bf16", M, D, draws(rng, "bf16", M, D)), Mat(lib, "bf16", D, N, draws(rng, "bf16", D, N))
        labels, out = Words(lib, rng.integers(0, N, M)), [Mat(lib, "f32", 1, M) for _ in range(4)]
        ops.Dropout(M, D, "bf16", 0.0, ld_y=ld).forward(x, p)  # spreads the rows out
        one, far = ops.CrossEntropy(M, D, N, "bf16"), ops.CrossEntropy(M, D, N, "bf16", ld_x=ld)
        ws, wb = Space(lib, one), Space(lib, one, True)
        one.forward(x, w, labels, out[0], lse=out[1], workspace=ws)
        far.forward(p, w, labels, out[2], lse=out[3], workspace=ws)
        assert np.array_equal(out[0].bits(), out[2].bits()) and np.array_equal(out[1].bits(), out[3].bits())
        dw = [Mat(lib, "bf16", D, N) for _ in range(2)]
        one.backward(x, w, labels, out[1], out[1], dw=dw[0], workspace=wb)
        far.backward(p, w, labels, out[1], out[1], dw=dw[1], workspace=wb)
        assert np.array_equal(dw[0].bits(), dw[1].bits())
        codes, s = [Mat(lib, "e4m3", M, D) for _ in range(2)], [Mat(lib, "f32", M, 1) for _ in range(2)]
        ops.Quantize(M, D, "bf16").forward(x, codes[0], s[0])
        ops.Quantize(M, D, "bf16", ld_x=ld).forward(p, codes[1], s[1])
        assert np.array_equal(codes[0].bits(), codes[1].bits()) and np.array_equal(s[0].bits(), s[1].bits())
        turned = [Mat(lib, "e4m3", D, M) for _ in range(2)]
        st = [Mat(lib, "f32", 1, 17) for _ in range(2)]
        ops.Quantize(M, D, "bf16", by="blocks").forward(x, turned[0], st[0])
        ops.Quantize(M, D, "bf16", by="blocks", ld_x=ld).forward(p, turned[1], st[1])
        assert np.array_equal(turned[0].bits(), turned[1].bits())
        o = [Mat(lib, "bf16", M, D) for _ in range(2)]
        near, wide = ops.Muon(M, D, "bf16"), ops.Muon(M, D, "bf16", ld_u=ld)
        wm = Space(lib, _NoDirection(near))
        near.orthogonalize(x, o[0], workspace=wm)
        wide.orthogonalize(p, o[1], workspace=wm)
        assert np.array_equal(o[0].bits(), o[1].bits())
        # codes and the result of their product in the large matrix
        w8, sw = Mat(lib, "e4m3", N, D), Mat(lib, "f32", 1, 1)
        ops.Quantize(D, N, "bf16", by="blocks").forward(w, w8, sw)
        y, back = Mat(lib, "bf16", M, N), Mat(lib, "bf16", M, N)
        ops.Linear8(M, D, N).forward(codes[0], s[0], w8, sw, y)
        ops.Linear8(M, D, N, ld_y=ld).forward(codes[0], s[0], w8, sw, p)
        ops.Dropout(M, N, "bf16", 0.0, ld_x=ld).forward(p, back)
        assert np.array_equal(y.bits(), back.bits())
    finally:
        lib.lib.volta_hip_device_free(p)


@pytest.mark.parametrize("t", TYPES)
def test_one_misaligned_matrix_among_aligned_ones(lib, t):
    """Rows of whole 16-byte chunks, one matrix an element off at a time: the
    results of the aligned call (whole numbers' sums are exact, so they do not
    depend on the form that the product takes)."""
    M, K, C_ = 80, 64, 96
    rng = np.random.default_rng(4)
    x, w = rng.integers(-2, 3, (M, K)) / 8.0, rng.integers(-2, 3, (K, C_)) / 8.0
    labels, dl = Words(lib, rng.integers(0, C_, M)), Mat(lib, "f32", 1, M, np.ones(M))
    op = ops.CrossEntropy(M, K, C_, t)
    ws, wb = Space(lib, op), Space(lib, op, True)
    want = None
    for off in ("", "x", "w", "dx", "dw"):
        say(t, "off:", off)
        m = {k: Mat(lib, t, *v.shape, v, lead=int(off == k)) for k, v in (("x", x), ("w", w))}
        out = {k: Mat(lib, t, *s, lead=int(off == k)) for k, s in (("dx", (M, K)), ("dw", (K, C_)))}
        loss, lse = Mat(lib, "f32", 1, M), Mat(lib, "f32", 1, M)
        op.forward(m["x"], m["w"], labels, loss, lse=lse, workspace=ws)
        if want:
            spoil(lib, lse)
            put(lib, lse, want[1].view(np.float32))  # the same lse: tiles differ in the order of its sum
        op.backward(m["x"], m["w"], labels, lse, dl, dx=out["dx"], dw=out["dw"], workspace=wb)
        got = [loss.get(), lse.bits(), out["dx"].get(), out["dw"].get()]
        if want is None:
            want = got
            continue
        assert np.abs(got[0] - want[0]).max() <= 2.0**-19
        for a, b in zip(got[2:], want[2:]):  # dz is the same; its products' sums have other orders
            assert np.abs(a - b).max() <= 2.0**-7 * np.abs(b).max()


def test_misaligned_codes(lib):
    """The product of codes from rows one byte off: the aligned one's, exactly
    (whole numbers and scales of powers of two)."""
    M, K, N = 70, 256, 144
    rng = np.random.default_rng(6)
    whole = encode(np.arange(-8, 9))
    x, w = rng.choice(whole, (M, K)), rng.choice(whole, (N, K))
    sx, sw = Mat(lib, "f32", M, 2, 2.0 ** rng.integers(-2, 3, (M, 2))), Mat(lib, "f32", 2, 2, 2.0 ** rng.integers(-2, 3, (2, 2)))
    op = ops.Linear8(M, K, N, "f32")
    ws, want = Space(lib, _NoDirection(op)), None
    for ox, ow in ((0, 0), (1, 0), (0, 1), (5, 3)):
        y = Mat(lib, "f32", M, N)
        op.forward(code_matrix(lib, x, lead=ox), sx, code_matrix(lib, w, lead=ow), sw, y, workspace=ws)
        want = y.bits() if want is None else want
        assert np.array_equal(y.bits(), want)
