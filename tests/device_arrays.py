"""Device arrays of the library's buffers for GPU tests: f32, f16 and bf16
values held as numpy holds them (bf16 as its bits), and captured graphs."""
import ctypes as C

import numpy as np

import willamette_hip as wh

HOST = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def to_kind(x, kind):
    """Rounded to nearest even from f32 (bf16: its upper 16 bits)."""
    x = np.asarray(x, np.float32)
    if kind != "bf16":
        with np.errstate(over="ignore"):
            return x.astype(HOST[kind])
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_kind(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


class Array:
    """A numpy array's copy on the device; `kind` says how its values are read."""

    def __init__(self, ctx, a, kind=None):
        a = np.ascontiguousarray(a)
        self.ctx, self.shape, self.dtype, self.kind = ctx, a.shape, a.dtype, kind
        self.buf = ctx.to_device(a) if a.size else ctx.alloc(16)

    @classmethod
    def full(cls, ctx, shape, value, kind):
        return cls(ctx, np.full(shape, to_kind(value, kind)), kind)

    @property
    def ptr(self):
        return self.buf.ptr

    def put(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        assert a.shape == self.shape
        self.ctx.check(wh.lib.wm_memcpy_h2d(self.ctx.h, self.buf.ptr, a.ctypes.data, a.nbytes))

    def host(self):
        """Behind the context's work."""
        out = np.empty(self.shape, self.dtype)
        if out.size:
            self.ctx.check(wh.lib.wm_memcpy_d2h(self.ctx.h, out.ctypes.data, self.buf.ptr, out.nbytes))
        return out

    def values(self):
        return from_kind(self.host(), self.kind)


def typed(ctx, rng, shape, kind, size=1.0):
    """Normal values of a type: on the device, and in 64 bits."""
    a = to_kind(rng.standard_normal(shape) * size, kind)
    return Array(ctx, a, kind), from_kind(a, kind)


def _hip():
    """The HIP runtime the library itself is linked to."""
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    return C.CDLL(path)


class Graph:
    """What `call` enqueues on the context's stream, captured."""

    def __init__(self, ctx, call):
        self.hip, self.stream = _hip(), C.c_void_p(ctx.stream)
        graph, self.exe = C.c_void_p(), C.c_void_p()
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 1))  # thread-local mode
        try:
            call()
        finally:
            st = self.hip.hipStreamEndCapture(self.stream, C.byref(graph))
        self._ok(st)
        self._ok(self.hip.hipGraphInstantiate(C.byref(self.exe), graph, None, None, C.c_size_t(0)))
        self._ok(self.hip.hipGraphDestroy(graph))

    @staticmethod
    def _ok(st):
        assert st == 0, f"hip error {st}"

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exe, self.stream))

    def close(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exe))
