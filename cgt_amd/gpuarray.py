"""Device arrays: the Python-side handle of a cgtArray with devtype GPU.

A GpuArray owns (or views) a contiguous row-major buffer in HBM, allocated
through the library's own cgt_amd_alloc -- the role cgtArray plays in the
reference with cgt_alloc (include/cgt_common.h:91-146, src/cgt_common.cpp:15-66).
Copies to and from numpy are synchronous, like the reference's cgt_memcpy.
"""
import numpy as np

from . import capi

# int8 is the reference's "i1" (what comparisons produce); float64 buffers exist
# only so tests can hand double data to checker kernels
_DTYPES = (np.dtype(np.float32), np.dtype(np.int32), np.dtype(np.int64), np.dtype(np.float64), np.dtype(np.int8))


class _Buffer(object):
    """Owns one device allocation; freed when the last array using it dies."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        self.ptr = capi.lib().cgt_amd_alloc(self.nbytes)
        if not self.ptr:
            raise capi.CgtAmdError("device allocation of %d bytes failed: %s"
                                   % (self.nbytes, capi.last_error()))

    def __del__(self):
        ptr = getattr(self, "ptr", None)
        if ptr and capi._LIB is not None:
            capi._LIB.cgt_amd_free(ptr)
            self.ptr = None


class GpuArray(object):
    def __init__(self, shape, dtype=np.float32, _buffer=None, _offset=0):
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        if self.dtype not in _DTYPES:
            raise TypeError("unsupported device dtype %s" % self.dtype)
        self.size = int(np.prod(self.shape, dtype=np.int64)) if self.shape else 1
        self.nbytes = self.size * self.dtype.itemsize
        self._buffer = _buffer if _buffer is not None else _Buffer(self.nbytes)
        self._offset = _offset
        assert self._offset + self.nbytes <= self._buffer.nbytes

    @property
    def ndim(self):
        return len(self.shape)

    @property
    def ptr(self):
        """Device address as an int (pass to the C ABI as void*)."""
        return self._buffer.ptr + self._offset

    @property
    def writeable(self):
        """False for a view of another library's read-only array: it is an input, never a result."""
        return getattr(self._buffer, "writeable", True)

    def check_writeable(self):
        if not self.writeable:
            raise ValueError("the array %r is another library's and read-only" % self)

    @property
    def __cuda_array_interface__(self):
        """Lets another library view this array without a copy."""
        return {"shape": self.shape, "typestr": self.dtype.str, "data": (self.ptr, not self.writeable), "strides": None, "version": 2}

    def reshape(self, *shape):
        """Zero-copy view with a new shape (the reference's Reshape op is a view
        too, cgt/core.py:1452-1465)."""
        if len(shape) == 1 and isinstance(shape[0], (tuple, list)):
            shape = tuple(shape[0])
        n = int(np.prod(shape, dtype=np.int64)) if shape else 1
        if n != self.size:
            raise ValueError("cannot reshape %s into %s" % (self.shape, shape))
        return GpuArray(shape, self.dtype, _buffer=self._buffer, _offset=self._offset)

    def set(self, host):
        self.check_writeable()
        host = _contiguous(host, self.dtype)
        if host.shape != self.shape:
            raise ValueError("shape mismatch %s vs %s" % (host.shape, self.shape))
        capi.check(capi.lib().cgt_amd_memcpy(capi.GPU, capi.CPU, self.ptr, host.ctypes.data, self.nbytes))
        return self

    def get(self):
        out = np.empty(self.shape, self.dtype)
        capi.check(capi.lib().cgt_amd_memcpy(capi.CPU, capi.GPU, out.ctypes.data, self.ptr, self.nbytes))
        return out

    def fill_u32(self, word, stream=None):
        self.check_writeable()
        capi.check(capi.lib().cgt_amd_fill_u32(self.ptr, word, self.nbytes // 4, stream))
        return self

    def __repr__(self):
        return "GpuArray(shape=%s, dtype=%s)" % (self.shape, self.dtype)


def empty(shape, dtype=np.float32):
    return GpuArray(shape, dtype)


class _Borrowed(object):
    """Device memory that belongs to another library's array, kept alive by holding on to it."""

    def __init__(self, ptr, nbytes, owner, writeable=True):
        self.ptr, self.nbytes, self.owner, self.writeable = ptr, nbytes, owner, writeable


def as_gpuarray(x):
    """Zero-copy view of another library's device array (anything with `__cuda_array_interface__`, e.g. a torch
    tensor on this GPU): contiguous, of a type device arrays have.  Calls made with it must be ordered with the
    other library's work by the caller (the same stream, or synchronisation).  A read-only array stays one: it is
    refused where a result is to be written.  Both libraries have to share one HIP
    runtime: import torch before the first call into this package."""
    if isinstance(x, GpuArray):
        return x
    info = x.__cuda_array_interface__
    dtype, shape = np.dtype(info["typestr"]), tuple(int(s) for s in info["shape"])
    if dtype not in _DTYPES:
        raise TypeError("unsupported device dtype %s" % dtype)
    strides = info.get("strides")
    if strides is not None and 0 not in shape:
        dense = dtype.itemsize
        for extent, stride in zip(reversed(shape), reversed(strides)):
            if extent > 1 and stride != dense:
                raise ValueError("device arrays are contiguous: shape %s with strides %s is not" % (shape, tuple(strides)))
            dense *= extent
    ptr = int(info["data"][0])
    if ptr == 0 and 0 not in shape:
        raise ValueError("the array has no device memory")
    if ptr % dtype.itemsize:
        raise ValueError("the array is not aligned to its elements")
    nbytes = int(np.prod(shape, dtype=np.int64)) * dtype.itemsize if shape else dtype.itemsize
    return GpuArray(shape, dtype, _buffer=_Borrowed(ptr, nbytes, x, writeable=not info["data"][1]))


def _contiguous(host, dtype=None):
    """C-contiguous copy/view that keeps 0-d arrays 0-d (np.ascontiguousarray makes them 1-d)."""
    host = np.asarray(host, dtype=dtype)
    return host if host.ndim == 0 else np.ascontiguousarray(host)


def to_gpu(host, dtype=None):
    host = _contiguous(host, dtype)
    return GpuArray(host.shape, host.dtype).set(host)
