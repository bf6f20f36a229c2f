"""Device memory, streams and graphs for tests of the operators that take device
pointers: the HIP runtime that libsp_hipkv.so itself uses, through ctypes."""
import ctypes

import numpy as np

import spkv

_hip = None


def hip():
    global _hip
    if _hip is None:
        spkv.kv()                                       # loads the runtime the library links
        _hip = ctypes.CDLL("libamdhip64.so.7")
        _hip.hipGetErrorString.restype = ctypes.c_char_p
    return _hip


def ok(rc):
    assert rc == 0, hip().hipGetErrorString(rc).decode()


class Dev:
    """A device copy of a numpy array."""

    def __init__(self, a):
        self.a = np.ascontiguousarray(a)
        self.p = ctypes.c_void_p()
        ok(hip().hipMalloc(ctypes.byref(self.p), ctypes.c_size_t(max(self.a.nbytes, 256))))
        self.put(self.a)

    def put(self, a):
        a = np.ascontiguousarray(a, dtype=self.a.dtype)
        assert a.nbytes == self.a.nbytes
        ok(hip().hipMemcpy(self.p, spkv.ptr(a), ctypes.c_size_t(a.nbytes), 1))
        ok(hip().hipDeviceSynchronize())

    @property
    def at(self):
        return self.p.value

    def get(self):
        out = np.empty_like(self.a)
        ok(hip().hipDeviceSynchronize())
        ok(hip().hipMemcpy(spkv.ptr(out), self.p, ctypes.c_size_t(out.nbytes), 2))
        return out

    def __del__(self):
        if self.p and _hip:
            _hip.hipFree(self.p)


def sync():
    ok(hip().hipDeviceSynchronize())


class Stream:
    def __init__(self):
        self.h = ctypes.c_void_p()
        ok(hip().hipStreamCreateWithFlags(ctypes.byref(self.h), 1))     # does not wait for the null stream

    def capture(self, f):
        """f(stream) recorded: returns an executable graph."""
        g, e = ctypes.c_void_p(), ctypes.c_void_p()
        ok(hip().hipStreamBeginCapture(self.h, 1))
        f(self.h.value)
        ok(hip().hipStreamEndCapture(self.h, ctypes.byref(g)))
        ok(hip().hipGraphInstantiate(ctypes.byref(e), g, None, None, ctypes.c_size_t(0)))
        ok(hip().hipGraphDestroy(g))
        return e

    def launch(self, e):
        ok(hip().hipGraphLaunch(e, self.h))

    def sync(self):
        ok(hip().hipStreamSynchronize(self.h))
