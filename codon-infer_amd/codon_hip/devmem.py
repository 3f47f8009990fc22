"""Device memory for callers of the CIH_IO_DEVICE forward, through
libamdhip64 directly (no torch): allocate, copy, free.  The forward itself
never needs this module; it is the plumbing a caller that keeps tokens and
outputs in HBM (the benchmark, the device-I/O tests) uses.
"""
import ctypes

import numpy as np

H2D, D2H, D2D = 1, 2, 3


class Hip:
    """Minimal device-memory plumbing through libamdhip64."""

    def __init__(self):
        self.L = ctypes.CDLL("libamdhip64.so")
        self.L.hipMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
        self.L.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
        self.L.hipMemset.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t]
        self.L.hipFree.argtypes = [ctypes.c_void_p]

    def malloc(self, n):
        p = ctypes.c_void_p()
        if self.L.hipMalloc(ctypes.byref(p), max(int(n), 1)) != 0:
            raise RuntimeError("hipMalloc failed")
        return p.value

    def h2d(self, dst, arr):
        if self.L.hipMemcpy(ctypes.c_void_p(dst), arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes, H2D) != 0:
            raise RuntimeError("hipMemcpy H2D failed")

    def d2h(self, arr, src):
        if self.L.hipMemcpy(arr.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(src), arr.nbytes, D2H) != 0:
            raise RuntimeError("hipMemcpy D2H failed")

    def d2d(self, dst, src, nbytes):
        if self.L.hipMemcpy(ctypes.c_void_p(dst), ctypes.c_void_p(src), nbytes, D2D) != 0:
            raise RuntimeError("hipMemcpy D2D failed")

    def memset(self, dst, value, nbytes):
        if self.L.hipMemset(ctypes.c_void_p(dst), value, nbytes) != 0:
            raise RuntimeError("hipMemset failed")

    def sync(self):
        self.L.hipDeviceSynchronize()

    def free(self, p):
        self.L.hipFree(ctypes.c_void_p(p))


class DeviceArray:
    """A row-major array in device memory, as the device operators take them
    (codon_hip.ops; torch tensors on the GPU serve as well): data_ptr(), shape,
    stride() in elements and dtype.  dtype is a numpy type, or "bfloat16" with
    the bits held as uint16 on the host."""

    def __init__(self, hip, values, dtype=None):
        a = np.ascontiguousarray(values)
        self._hip, self._np = hip, a.dtype
        self.dtype = dtype or a.dtype.name
        self.shape = a.shape
        self._ptr = hip.malloc(a.nbytes)
        if a.nbytes:
            hip.h2d(self._ptr, a)

    def data_ptr(self):
        return self._ptr

    def stride(self):
        st, n = [], 1
        for d in reversed(self.shape):
            st.append(n)
            n *= max(d, 1)
        return tuple(reversed(st))

    def numpy(self):
        """The values (after what was enqueued before has run)."""
        a = np.empty(self.shape, self._np)
        self._hip.sync()
        if a.nbytes:
            self._hip.d2h(a, self._ptr)
        return a

    def free(self):
        if self._ptr:
            self._hip.free(self._ptr)
            self._ptr = 0
