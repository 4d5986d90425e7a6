"""Device buffers, streams and graphs for the operators' tests, through the HIP runtime."""
import ctypes as C

import numpy as np

from tests.harness import moe

TYPES = {"f32": moe.QT_F32, "f16": moe.QT_F16, "bf16": moe.QT_BF16}
RAW = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def encode(x, type):
    """Values rounded to type, as its raw elements (bf16: the upper half of fp32's bits, to nearest even)."""
    with np.errstate(over="ignore"):
        x = np.ascontiguousarray(x, dtype=np.float32)
        if type != "bf16":
            return x.astype(RAW[type])
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(a, type):
    if type == "bf16":
        a = (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float64)


class Buf:
    """A device buffer holding an array."""

    def __init__(self, hip, a):
        self.hip, self.shape, self.dtype, self.nbytes = hip, a.shape, a.dtype, a.nbytes
        p = C.c_void_p()
        assert hip.rt.hipMalloc(C.byref(p), max(a.nbytes, 256)) == 0
        self.ptr = p.value
        self.put(a)

    def put(self, a, at=0):
        a = np.ascontiguousarray(a, dtype=self.dtype)
        assert at + a.nbytes <= max(self.nbytes, 256)
        assert self.hip.rt.hipMemcpy(self.ptr + at, a.ctypes.data, a.nbytes, 1) == 0

    def get(self, at=0, shape=None):
        """(Waits for the device.)"""
        a = np.empty(self.shape if shape is None else shape, self.dtype)
        assert self.hip.rt.hipDeviceSynchronize() == 0
        assert at + a.nbytes <= max(self.nbytes, 256)
        assert self.hip.rt.hipMemcpy(a.ctypes.data, self.ptr + at, a.nbytes, 2) == 0
        return a

    def free(self):
        if self.ptr:
            self.hip.rt.hipFree(self.ptr)
            self.ptr = None

    __del__ = free


class Raw(Buf):
    """A large buffer of bytes, all of one value."""

    def __init__(self, hip, n, value=0):
        self.hip, self.shape, self.dtype, self.nbytes = hip, (n,), np.dtype(np.uint8), n
        p = C.c_void_p()
        assert hip.rt.hipMalloc(C.byref(p), n) == 0
        self.ptr = p.value
        self.fill(value)

    def fill(self, value):
        assert self.hip.rt.hipMemset(self.ptr, value, self.nbytes) == 0
        assert self.hip.rt.hipDeviceSynchronize() == 0


class Hip:
    def __init__(self):
        self.rt = rt = C.CDLL("libamdhip64.so")
        P, N = C.c_void_p, C.c_size_t
        for name, args in (("hipMalloc", [C.POINTER(P), N]), ("hipFree", [P]), ("hipMemcpy", [P, P, N, C.c_int]),
                           ("hipMemset", [P, C.c_int, N]), ("hipDeviceSynchronize", []), ("hipStreamSynchronize", [P]),
                           ("hipStreamCreateWithFlags", [C.POINTER(P), C.c_uint]), ("hipStreamDestroy", [P]),
                           ("hipStreamBeginCapture", [P, C.c_int]), ("hipStreamEndCapture", [P, C.POINTER(P)]),
                           ("hipGraphInstantiate", [C.POINTER(P), P, P, P, N]), ("hipGraphLaunch", [P, P]),
                           ("hipGraphExecDestroy", [P]), ("hipGraphDestroy", [P])):
            getattr(rt, name).argtypes = args

    def put(self, a):
        return Buf(self, np.ascontiguousarray(a))

    def full(self, shape, value, dtype=np.float32):
        return Buf(self, np.full(shape, value, dtype))

    def rows(self, x, type, extra=0, behind=0, fill=np.nan):
        """x in type, its rows cols + extra apart and `behind` rows after the last, filled up with `fill`; and the values."""
        x = np.asarray(x, np.float32)
        a = encode(np.full((x.shape[0] + behind, x.shape[1] + extra), fill, np.float32), type)
        a[:x.shape[0], :x.shape[1]] = encode(x, type)
        return Buf(self, a), decode(a[:x.shape[0], :x.shape[1]], type)

    def stream(self):
        s = C.c_void_p()
        assert self.rt.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        return s.value

    def wait(self, stream):
        assert self.rt.hipStreamSynchronize(stream) == 0

    def capture(self, stream, calls):
        """The graph of what calls() enqueues on stream, as a function that launches it there."""
        g, x = C.c_void_p(), C.c_void_p()
        assert self.rt.hipStreamBeginCapture(stream, 1) == 0  # (this thread's calls)
        try:
            calls()
        finally:
            st = self.rt.hipStreamEndCapture(stream, C.byref(g))
        assert st == 0
        assert self.rt.hipGraphInstantiate(C.byref(x), g, None, None, 0) == 0
        return lambda: self.check(self.rt.hipGraphLaunch(x, stream))

    @staticmethod
    def check(st):
        assert st == 0


hip = Hip()
