"""What the operators' tests share: element types on the host, matrices in
device memory with guarded gaps, and the operators' definitions in 64 bits."""
from __future__ import annotations

import numpy as np

TYPES = ("f32", "bf16", "f16")
STORE = {"f32": np.float32, "bf16": np.uint16, "f16": np.float16, "e4m3": np.uint8}
NAN = {"f32": np.uint32(0x7FC0A001), "bf16": np.uint16(0x7FA1), "f16": np.uint16(0x7E21), "e4m3": np.uint8(0x7F)}
BITS = {"f32": np.uint32, "bf16": np.uint16, "f16": np.uint16, "e4m3": np.uint8}
# half a step of the type relative to the value, and half the step of its subnormals
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11, "e4m3": 2.0**-4}
FLOOR = {"f32": 2.0**-149, "bf16": 2.0**-133, "f16": 2.0**-25, "e4m3": 2.0**-10}
GELU_C, GELU_K = 0.7978845608, 0.044715


def pack(v, t):
    """Values rounded to the nearest of type t, as stored."""
    v32 = np.asarray(v, np.float32)
    if t == "f32":
        return v32
    if t == "f16":
        return v32.astype(np.float16)
    b = v32.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(v32), np.uint16(0x7FC0), r)


def unpack(s, t):
    """Stored values as float64."""
    if t == "bf16":
        return (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if t == "e4m3":
        c = s.astype(np.int64)
        e, m = (c >> 3) & 15, c & 7
        v = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
        return np.where((c & 127) == 127, np.nan, np.where(c >> 7, -v, v))
    return s.astype(np.float64)


class Mat:
    """A [rows x cols] matrix of type t in device memory with rows ld apart,
    `lead` elements into its allocation; everything around it holds a NaN
    pattern that must still be there afterwards."""

    def __init__(self, lib, t, rows, cols, values=None, ld=None, lead=0):
        from volta_amd import DeviceArray

        self.t, self.rows, self.cols, self.ld, self.lead = t, rows, cols, ld or cols, lead
        n = lead + max(rows, 1) * self.ld + 24
        host = np.full(n, NAN[t], BITS[t])
        if values is not None and rows:
            self._view(host)[:, :] = pack(values, t).reshape(rows, cols).view(BITS[t])
        self.before = host
        self.dev = DeviceArray(host, lib)
        self.ptr = self.dev.ptr + lead * host.itemsize

    def _view(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.lead:], (self.rows, self.cols),
                                               (self.ld * flat.itemsize, flat.itemsize))

    def bits(self):
        """What the device holds now; nothing outside the matrix may have changed."""
        flat = self.dev.numpy()
        mine = np.zeros(flat.size, bool)
        if self.rows:
            self._view(mine)[:, :] = True
        assert np.array_equal(flat[~mine], self.before[~mine]), "written outside the matrix"
        return self._view(flat).copy() if self.rows else np.zeros((0, self.cols), flat.dtype)

    def get(self):
        return unpack(self.bits().view(STORE[self.t]), self.t)

    def untouched(self):
        return np.array_equal(self.dev.numpy(), self.before)


def floats(lib, n):
    return Mat(lib, "f32", 1, max(n, 1))


def act(name, x):
    """f(x) and f'(x) by their definitions."""
    with np.errstate(over="ignore"):
        q = 1 / (1 + np.exp(-x))
    if name == "relu":
        return np.maximum(x, 0), (x > 0) * 1.0
    if name == "leaky_relu":
        return np.where(x > 0, x, 0.01 * x), np.where(x > 0, 1.0, 0.01)
    if name == "sigmoid":
        return q, q * (1 - q)
    if name == "tanh":
        return np.tanh(x), 1 - np.tanh(x) ** 2
    if name == "silu":
        return x * q, q + x * q * (1 - q)
    if name == "gelu":
        th = np.tanh(GELU_C * (x + GELU_K * x**3))
        return (0.5 * x * (1 + th),
                0.5 * (1 + th) + 0.5 * x * (1 - th * th) * GELU_C * (1 + 3 * GELU_K * x * x))
    return x, np.ones_like(x)


def act_error(t, x):
    """How far the kernels' f and f' may be off at x, beside the rounding of x
    itself.  16 bits: the hardware's exp2 and reciprocal are within 2^-23 of
    their result, the exponent's argument within 2^-23 of itself (|x| log2 e
    2^-23 of the result), tanh's series within 1.4e-5 of itself: 2e-5 of the
    result and 1e-6 for differences of such terms.  float32: eight roundings
    of terms no larger than 1 + |x|."""
    if t == "f32":
        e = 8 * HALF[t] * (1 + np.abs(x))
        return e, 2 * e
    e = 2e-5 * np.minimum(np.abs(x) + 1, 4) + 1e-6
    return e, e


def rounded(v, t):
    """The error of rounding v to type t."""
    return HALF[t] * np.abs(v) + FLOOR[t]


def held(v, t):
    """v, infinite where rounding to type t makes it so (float16 ends at 65504)."""
    return np.where(np.abs(v) >= 65520.0, np.copysign(np.inf, v), v) if t == "f16" else v


def check(got, want, tol, what):
    """Every value within its tolerance; says where it is furthest off."""
    assert got.shape == want.shape, f"{what}: shape {got.shape} against {want.shape}"
    if got.size == 0:
        return
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want) / tol
    off = np.where(got == want, 0, np.where(np.isnan(off), np.inf, off))
    i = np.unravel_index(np.argmax(off), off.shape)
    assert off[i] <= 1, (f"{what}: {got[i]} at {i}, should be {want[i]} within {np.broadcast_to(tol, off.shape)[i]} "
                         f"({np.mean(off > 1):.3%} of the values are outside)")


def splitmix_keep(n, seed, offset, p):
    """keep of elements 0 .. n-1 (whole-number arithmetic of Python)."""
    mask = (1 << 64) - 1
    out = np.zeros(n, bool)
    threshold = int(p * 2.0**32)
    for j in range((n + 1) // 2):
        z = (seed + (offset + j + 1) * 0x9E3779B97F4A7C15) & mask
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
        z ^= z >> 31
        for i, bits in ((2 * j, z & 0xFFFFFFFF), (2 * j + 1, z >> 32)):
            if i < n:
                out[i] = bits >= threshold
    return out
