"""A call captured into a graph and replayed, for the operators' tests."""
from __future__ import annotations

import ctypes as C

from tests import ops_ref as R


def hip(lib):
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


class Captured:
    """What `call(stream)` enqueues, captured once; a stream of its own."""

    def __init__(self, lib, call):
        self.hip = hip(lib)
        self.stream, self.graph, self.run = C.c_void_p(), C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamCreate(C.byref(self.stream)) == 0
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # thread-local
        call(self.stream.value)
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, 0) == 0

    def replay(self):
        assert self.hip.hipDeviceSynchronize() == 0
        assert self.hip.hipGraphLaunch(self.run, self.stream) == 0
        assert self.hip.hipStreamSynchronize(self.stream) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.run) == 0 and self.hip.hipGraphDestroy(self.graph) == 0
        assert self.hip.hipStreamDestroy(self.stream) == 0


def put(lib, m, values):
    """Other values into a Mat of ops_ref."""
    host = m.before.copy()
    m._view(host)[:, :] = R.pack(values, m.t).reshape(m.rows, m.cols).view(R.BITS[m.t])
    m.before = host
    assert lib.lib.volta_hip_copy(m.dev.ptr, host.ctypes.data, host.nbytes, 1) == 0


def spoil(lib, m):
    """What the Mat held before any call."""
    assert lib.lib.volta_hip_copy(m.dev.ptr, m.before.ctypes.data, m.before.nbytes, 1) == 0
