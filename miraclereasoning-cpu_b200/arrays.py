"""Device arrays of several types and owners, for the operators that take more than float32 buffers.

An operator argument is a backend ``Tensor`` (float32), a ``DeviceArray`` made by ``CUDABackend.upload_array`` /
``empty_array``, or any object with the same accessors on the backend's GPU: ``data_ptr()``, ``shape``, ``stride()``,
``dtype`` (named float32, float16, bfloat16 or int32), ``get_device()`` and ``new_empty(shape)``, as torch tensors
have.  The owner keeps the memory alive until the queued work is done.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import math
import struct
from pathlib import Path

import numpy as np

from . import _native
from .weights import float32_to_bf16_bits

TYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "int32": 3}   # enum mr_dtype
_ITEM = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4}
_CODES = {}    # a dtype object -> its code, as its name says


def described(array, name, device):
    """The mr_array of an operator's argument, as bytes; ValueError if it is none on the device.  (_pycall reads
    the usual ones itself and comes here for a type's first array, and for those that are wrong.)"""
    for accessor in ("get_device", "data_ptr", "stride", "shape", "dtype"):
        if not hasattr(array, accessor):
            raise ValueError(f"{name} must be a device array, not {type(array).__name__}")
    where, shape, dtype = array.get_device(), tuple(array.shape), array.dtype
    if where != device:
        raise ValueError(f"{name} must be on device {device}, not {where if where >= 0 else 'the host'}")
    if not 0 < len(shape) < 5:
        raise ValueError(f"{name} must have 1 to 4 dimensions, not {len(shape)}")
    code = TYPES.get(str(dtype).rsplit(".", 1)[-1])
    if code is None:
        raise ValueError(f"unsupported array type {dtype}: float32, float16, bfloat16 or int32 is needed")
    _CODES[dtype] = code
    pad = (0,) * (4 - len(shape))
    return struct.pack("<Qii8q", array.data_ptr(), code, len(shape), *shape, *pad, *array.stride(), *pad)


# the operators in csrc/pycall.c's order
APPEND, PAGED, WINDOW, EVICT = range(4)
_NAMES = ("mr_append_pages", "mr_paged_attention", "mr_window_attention", "mr_evict_pages")
# this interpreter's own build of csrc/pycall.c
PYCALL = Path(__file__).resolve().with_name("_pycall" + importlib.machinery.EXTENSION_SUFFIXES[0])
_module = None   # the module, once a call has needed it
_call = None     # its call(), once the library's operators are handed over to it


def _pycall():
    global _module
    if _module is None:
        try:
            spec = importlib.util.spec_from_file_location(f"{__package__}._pycall", PYCALL)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as missing:
            raise _native.CUDAError(f"{PYCALL} is missing or unusable ({missing}): build it with "
                                    f"'python miraclereasoning-cpu_b200/build.py'") from None
        module.types(_CODES, described)
        _module = module
    return _module


def describe(array, name, device):
    """An operator's argument as mr_array, in bytes."""
    return _pycall().describe(array, name, device)


def _bound():
    global _call
    lib, module = _native.library(), _pycall()
    module.bind(*[C.cast(getattr(lib, name), C.c_void_p).value for name in _NAMES])
    _call = module.call
    return _call


def invoke(which, *args):
    """An operator: its context's address, the device, arrays (None: left out) and scalars."""
    status = (_call or _bound())(which, *args)
    if status:
        _native.check(status, _NAMES[which])


class DeviceArray:
    """Contiguous device memory of one type, owned by the library and freed on __del__."""

    def __init__(self, backend, shape, dtype):
        shape = (shape,) if isinstance(shape, int) else tuple(shape)
        if not shape or any(not isinstance(n, int) or n < 0 for n in shape):
            raise ValueError(f"invalid array shape: {shape}")
        if dtype not in TYPES:
            raise ValueError(f"unsupported array type {dtype}: float32, float16, bfloat16 or int32 is needed")
        self.backend, self.shape, self.dtype = backend, shape, dtype
        self.size = math.prod(shape)
        self.words = max(1, -(-self.size * _ITEM[dtype] // 4))   # the buffer's float32 elements
        handle, pointer = C.c_void_p(), C.c_void_p()
        _native.call("mr_buffer_alloc", backend.context, self.words, C.byref(handle))
        self.handle = handle.value
        _native.call("mr_buffer_pointer", self.handle, C.byref(pointer))
        self._pointer = pointer.value

    def __del__(self):
        handle = getattr(self, "handle", None)
        if handle and _native._lib is not None:
            _native._lib.mr_buffer_free(handle)
            self.handle = None

    def data_ptr(self):
        return self._pointer

    def get_device(self):
        return self.backend.device.ordinal

    def stride(self):
        strides, step = [], 1
        for n in reversed(self.shape):
            strides.append(step)
            step *= max(n, 1)
        return tuple(reversed(strides))

    def new_empty(self, shape):
        return DeviceArray(self.backend, shape, self.dtype)


def stored(array, dtype):
    """A host array as `dtype` stores it (bfloat16: the bits, rounded to nearest even)."""
    if dtype == "bfloat16":
        return float32_to_bf16_bits(np.ascontiguousarray(array, dtype=np.float32))
    return np.ascontiguousarray(array, dtype=dtype)


def widened(raw, dtype):
    return (raw.astype(np.uint32) << np.uint32(16)).view(np.float32) if dtype == "bfloat16" else raw


def host_type(dtype):
    return np.dtype(np.uint16 if dtype == "bfloat16" else dtype)
