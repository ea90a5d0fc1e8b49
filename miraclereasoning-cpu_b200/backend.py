"""``CUDABackend``: the reference backend's method surface on a B200.

Drop-in for ``OpenCLBackend`` (miracle_reasoning/opencl.py:129-303): the same
``empty/upload/read/copy/run/linear/norm/rotate/add/swiglu/softmax/attention/
mix/finish`` methods with the same argument meaning, shapes and error
behaviour, and a ``device`` with ``max_allocation_bytes`` and ``to_dict()``.
Tensors are float32 device buffers owned by the C library; ``run(name, ...)``
dispatches to the kernel's ``mr_op_*`` entry point.  There is no host fallback:
a missing library or device raises ``CUDAError``.

Beyond the reference: a paged key / value cache for serving several sequences
(``append_pages``, ``append_rotated``, ``read_pages``, ``paged_attention``,
``window_attention``, ``evict_pages``), and ``log_probabilities`` of its logits,
on arrays of any owner in float32, float16 or bfloat16 (``arrays.py``); the cache
may be held in 4 bits a value.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import numpy as np

from . import _native, arrays
from ._native import CUDAError, call
from .arrays import DeviceArray, empty_like, host_type, invoke, stored, widened

# kernel name -> (NDRange rank, argument kinds) in kernels.cl order
_KERNELS = {
    "linear": (2, "pppiii"), "rms": (1, "pppiifi"), "rope": (1, "ppppiiii"), "swiglu": (1, "pppi"),
    "axpy": (1, "pppif"), "scores": (2, "ppppiiiiiii"), "softmax": (1, "ppii"),
    "latent_mask": (2, "ppiiii"), "mix": (1, "ppppiiiiiii"), "pool_scores": (2, "pppiii"),
    "pool_mix": (2, "ppppiiii"), "merge_rows": (1, "ppiff"), "block_means": (2, "ppiii"),
}
_KIND_NAMES = {"p": "a tensor", "i": "an int", "f": "a float"}


@dataclass(frozen=True)
class Device:
    ordinal: int
    name: str
    kind: str
    memory_bytes: int
    max_allocation_bytes: int
    sm_count: int
    compute_capability: str

    def to_dict(self):
        return dict(vars(self))


def list_devices():
    """CUDA devices visible to this process ([] when there is none)."""
    lib = _native.library()
    count = C.c_int()
    _native.check(lib.mr_device_count(C.byref(count)), "mr_device_count")
    devices = []
    for i in range(count.value):
        info = _native.DeviceInfo()
        _native.check(lib.mr_device_query(i, C.byref(info)), "mr_device_query")
        devices.append(Device(i, info.name.decode(), "gpu", int(info.memory_bytes),
                              int(info.max_allocation_bytes), info.sm_count, f"{info.cc_major}.{info.cc_minor}"))
    return devices


class Tensor:
    """float32 device buffer (reference Tensor: shape, size, handle; freed on __del__)."""

    def __init__(self, backend, handle, shape):
        self.backend, self.handle, self.shape = backend, handle, tuple(shape)
        self.size = math.prod(self.shape)

    def __del__(self):
        handle = getattr(self, "handle", None)
        if handle and _native._lib is not None:
            _native._lib.mr_buffer_free(handle)
            self.handle = None

    # the accessors of an operator's array argument (arrays.py)
    dtype = "float32"
    stride = DeviceArray.stride
    get_device = DeviceArray.get_device

    def data_ptr(self):
        pointer = C.c_void_p()
        call("mr_buffer_pointer", self.handle, C.byref(pointer))
        return pointer.value

    def new_empty(self, shape, dtype="float32"):
        return self.backend.empty(shape) if dtype == "float32" and all(shape) else DeviceArray(self.backend, shape, dtype)


def _count(value, name, least=0):
    if type(value) is int and least <= value < 2 ** 31:
        return value
    if isinstance(value, np.integer) and least <= value < 2 ** 31:
        return int(value)
    raise ValueError(f"{name} must be a whole number from {least} on{', or None' if least else ''}: {value!r}")


def _no_array(array, name):
    return ValueError(f"{name} must be a device array, not {type(array).__name__}")


def _like(array, name):
    try:
        return array.new_empty(array.shape)
    except AttributeError:
        raise _no_array(array, name) from None


class CUDABackend:
    """Float32 execution on one B200 (one context = one device + one stream).

    ``stream``: a CUDA stream of the caller's (its handle as an int; 0 is the
    legacy default stream) on which all of this backend's work is queued, in
    order with the caller's own; it has to outlive the backend.  None: a stream
    of its own, which the caller orders with other streams' work (``finish``).

    An instance must be used by a single thread at a time, as the reference
    backend requires.
    """

    def __init__(self, *, device_index=0, platform_index=None, device_type="gpu", stream=None):
        if device_type not in ("gpu", "cuda"):
            raise ValueError("CUDABackend executes on a CUDA GPU; device_type must be 'gpu'")
        devices = list_devices()
        if not 0 <= device_index < len(devices):
            raise CUDAError(f"No CUDA device {device_index} (found {len(devices)}); no automatic CPU fallback.")
        self.device = devices[device_index]
        handle = C.c_void_p()
        if stream is None:
            call("mr_context_create", device_index, C.byref(handle))
        else:
            call("mr_context_create_on_stream", device_index, stream, C.byref(handle))
        self.context = handle
        self._where = handle.value, device_index   # of every array operator's call

    def __del__(self):
        ctx = getattr(self, "context", None)
        if ctx and _native._lib is not None:
            _native._lib.mr_context_destroy(ctx)
            self.context = None

    # buffers (opencl.py:178-217) -------------------------------------------------
    def empty(self, shape):
        shape = tuple(shape)
        if not shape or any(not isinstance(n, int) or n <= 0 for n in shape):
            raise ValueError(f"invalid tensor shape: {shape}")
        size = math.prod(shape) * 4
        if size > self.device.max_allocation_bytes:
            raise CUDAError(f"Buffer needs {size:,} bytes, above device allocation limit "
                            f"{self.device.max_allocation_bytes:,}; reduce context or weight tile size")
        handle = C.c_void_p()
        call("mr_buffer_alloc", self.context, math.prod(shape), C.byref(handle))
        return Tensor(self, handle.value, shape)

    def upload(self, array):
        array = np.ascontiguousarray(array, dtype=np.float32)
        out = self.empty(array.shape)
        call("mr_buffer_upload", out.handle, 0, array.ctypes.data, array.size)
        return out

    def read(self, tensor):
        self._owns(tensor)
        out = np.empty(tensor.shape, dtype=np.float32)
        call("mr_buffer_download", tensor.handle, 0, out.ctypes.data, out.size)
        return out

    def _owns(self, *tensors):
        if any(t.backend is not self for t in tensors):
            raise ValueError("Tensors belong to different CUDA contexts")

    def copy(self, source, target, *, source_offset=0, target_offset=0, count=None):
        self._owns(source, target)
        count = source.size - source_offset if count is None else count
        if (min(source_offset, target_offset, count) < 0 or source_offset + count > source.size
                or target_offset + count > target.size):
            raise ValueError("tensor copy is out of bounds")
        if count:
            call("mr_buffer_copy", source.handle, target.handle, source_offset, target_offset, count)

    # dispatch (opencl.py:219-239) -------------------------------------------------
    def run(self, name, shape, *args):
        if name not in _KERNELS:
            raise CUDAError(f"create kernel {name} failed (no such kernel)")
        rank, kinds = _KERNELS[name]
        shape = tuple(int(s) for s in shape)
        if len(shape) != rank or len(args) != len(kinds):
            raise ValueError(f"{name}: NDRange rank or argument count mismatch")
        values = []
        for index, (arg, kind) in enumerate(zip(args, kinds)):
            if isinstance(arg, Tensor):
                self._owns(arg)
                value = C.c_void_p(arg.handle)
            elif isinstance(arg, (float, np.floating)):
                value = C.c_float(arg)
            elif isinstance(arg, (int, np.integer)) and -(2 ** 31) <= arg < 2 ** 31:
                value = C.c_int(arg)
            else:
                raise ValueError(f"unsupported kernel argument: {arg}")
            expected = {"p": C.c_void_p, "i": C.c_int, "f": C.c_float}[kind]
            if type(value) is not expected:
                if kind == "f" and isinstance(value, C.c_int):
                    value = C.c_float(value.value)
                else:
                    raise ValueError(f"{name}: argument {index} must be {_KIND_NAMES[kind]}")
            values.append(value)
        call(f"mr_op_{name}", self.context, *shape, *values)

    # op helpers, same launch geometry as opencl.py:241-300 ------------------------
    def linear(self, x, weight):
        if len(x.shape) != 2 or len(weight.shape) != 2 or x.shape[1] != weight.shape[1]:
            raise ValueError("linear needs x[rows,in] and weight[out,in]")
        rows, inner = x.shape
        out = self.empty((rows, weight.shape[0]))
        self.run("linear", (weight.shape[0], rows), x, weight, out, rows, weight.shape[0], inner)
        return out

    def norm(self, x, weight, width, eps):
        if x.size % width or (weight is not None and weight.shape != (width,)):
            raise ValueError("RMSNorm shape mismatch")
        out = self.empty(x.shape)
        self.run("rms", (x.size // width,), x, weight if weight is not None else x, out,
                 x.size // width, width, float(eps), int(weight is not None))
        return out

    def rotate(self, x, frequencies, positions, heads, dim, split_half=False):
        if x.shape != (positions.size, heads * dim):
            raise ValueError("RoPE shape mismatch")
        out = self.empty(x.shape)
        self.run("rope", (x.size // 2,), x, frequencies, positions, out, positions.size, heads, dim,
                 int(split_half))
        return out

    def add(self, x, y, scale=1.0):
        if x.shape != y.shape:
            raise ValueError("residual shapes differ")
        out = self.empty(x.shape)
        self.run("axpy", (x.size,), x, y, out, x.size, float(scale))
        return out

    def swiglu(self, gate, up):
        if gate.shape != up.shape:
            raise ValueError("SwiGLU shapes differ")
        out = self.empty(gate.shape)
        self.run("swiglu", (gate.size,), gate, up, out, gate.size)
        return out

    def softmax(self, x):
        out = self.empty(x.shape)
        self.run("softmax", (x.shape[0],), x, out, *x.shape)
        return out

    def attention(self, query, keys, values, *, heads, kv_heads, dim, start, length,
                  extra_keys=None, extra_values=None, extra_length=0):
        scores = self.empty((heads, length + extra_length))
        self.run("scores", (length + extra_length, heads), query, keys,
                 extra_keys if extra_keys is not None else keys, scores,
                 heads, kv_heads, dim, keys.shape[0], start, length, extra_length)
        return self.mix(self.softmax(scores), values, heads, kv_heads, dim, start, length,
                        extra_values, extra_length)

    def mix(self, probs, values, heads, kv_heads, dim, start, length, extra_values=None, extra_length=0):
        out = self.empty((1, heads * dim))
        self.run("mix", (heads * dim,), probs, values,
                 extra_values if extra_values is not None else values, out,
                 heads, kv_heads, dim, values.shape[0], start, length, extra_length)
        return out

    # arrays of other types (arrays.py) ---------------------------------------------
    def empty_array(self, shape, dtype="float32"):
        return DeviceArray(self, shape, dtype)

    def upload_array(self, array, dtype="float32"):
        """A host array on the device; bfloat16 rounds float values to nearest even."""
        raw = stored(array, dtype)
        out = DeviceArray(self, raw.shape, dtype)
        if out.size:
            flat = np.zeros(out.words, np.uint32)
            flat.view(np.uint8)[:raw.nbytes] = raw.reshape(-1).view(np.uint8)
            call("mr_buffer_upload", out.handle, 0, flat.ctypes.data, out.words)
        return out

    def read_array(self, array):
        """A DeviceArray's values on the host (bfloat16 widened to float32)."""
        self._owns(array)
        flat = np.empty(array.words, np.uint32)
        call("mr_buffer_download", array.handle, 0, flat.ctypes.data, array.words)
        kind = host_type(array.dtype)
        raw = flat.view(np.uint8)[:array.size * kind.itemsize].view(kind).reshape(array.shape)
        return widened(raw, array.dtype)

    # paged key / value cache (include/miracle_cuda.h: mr_array and what follows) -----
    # Pools are [pages, page rows, kv heads, dim], page_table [batch, table pages] and lengths
    # [batch] int32; row t of sequence s is row t % page rows of page page_table[s, t // page rows].
    # Pools of uint8 [pages, page rows, kv heads, 5 dim / 8] hold 4 bits a value, for head dims 32, 64, 96 and 128:
    # a step and a base for 32 values (the header has the format).  append_pages, append_rotated, read_pages,
    # paged_attention and evict_pages take them.

    def append_pages(self, keys, values, key_pages, value_pages, page_table, lengths, offsets=None):
        """New rows [tokens, kv heads, dim] into their pages.  ``lengths`` counts them already; sequence s's
        new rows are offsets[s] .. offsets[s + 1] - 1 (``offsets`` None: one row per sequence)."""
        invoke(arrays.APPEND, *self._where, keys, values, key_pages, value_pages, page_table, lengths, offsets)

    def append_rotated(self, keys, values, key_pages, value_pages, page_table, lengths, frequencies, offsets=None, *,
                       positions=None, query=None, out=None, split_half=False):
        """``append_pages`` with the position rotation on the way: the first 2 n dims of ``keys``, and of ``query``
        [tokens, heads, dim], are turned by position * ``frequencies`` [n] (float32), in pairs of neighbours or with
        ``split_half`` of dims p and p + n (as ``rotate`` does).  ``positions`` int32 [tokens]; None: a token's row of
        its sequence.  Returns the turned query, ``out`` (an array like the query, of memory that none of the others
        has; rows of no sequence are not written), or None without one."""
        if query is not None and out is None:
            out = _like(query, "query")
        invoke(arrays.ROTATED, *self._where, query, keys, values, key_pages, value_pages, page_table, lengths, offsets,
               frequencies, positions, out, 1 if split_half else 0)
        return out

    def read_pages(self, key_pages, value_pages, page_table, lengths, offsets, keys, values):
        """The way back of ``append_pages``: each sequence's last rows from their pages to ``keys`` and ``values``
        [tokens, kv heads, dim], sequence s's to offsets[s] .. offsets[s + 1] - 1 (``offsets`` None: its newest row
        alone).  From 4-bit pages as any floating type, so that ``window_attention`` can take a prompt's later part.
        Rows that no page holds are zeros.  Returns (keys, values)."""
        invoke(arrays.READ, *self._where, key_pages, value_pages, page_table, lengths, offsets, keys, values)
        return keys, values

    def paged_attention(self, query, key_pages, value_pages, page_table, lengths, *, window=None, sinks=0, scale=None,
                        weights=None, out=None):
        """Attention of every sequence's newest token, query [batch, heads, dim], over its rows; returns ``out``
        (an array like the query).  ``window``: only the newest rows, and the first ``sinks``, are visible.
        ``scale`` defaults to 1 / sqrt(dim).  ``weights`` float32 [batch, kv heads, table rows] has each row's
        softmax weights, summed over the query heads that share its head, added to it."""
        window = 0 if window is None else _count(window, "window", 1)
        if out is None:
            out = _like(query, "query")
        invoke(arrays.PAGED, *self._where, query, key_pages, value_pages, page_table, lengths, weights, out, window,
               _count(sinks, "sinks"), query.shape[-1] ** -0.5 if scale is None else scale)
        return out

    def window_attention(self, query, keys, values, query_offsets, key_offsets=None, *, window=None, sinks=0,
                         scale=None, out=None):
        """Causal attention of prompts packed one after the other: query [tokens, heads, dim], keys and values
        [rows, kv heads, dim], sequence s's rows at query_offsets[s] .. query_offsets[s + 1] - 1 and at
        ``key_offsets`` (None: the same) alike; its last query stands at its last key.  A query sees the newest
        ``window`` keys up to its own (None: all) and the first ``sinks``.  Returns ``out`` (an array like the
        query; rows of no sequence are not written)."""
        window = 0 if window is None else _count(window, "window", 1)
        if out is None:
            out = _like(query, "query")
        invoke(arrays.WINDOW, *self._where, query, keys, values, query_offsets,
               query_offsets if key_offsets is None else key_offsets, out, window, _count(sinks, "sinks"),
               query.shape[-1] ** -0.5 if scale is None else scale)
        return out

    def evict_pages(self, key_pages, value_pages, page_table, lengths, weights, target_table, *, budget, sinks=0,
                    recent=0, target_keys=None, target_values=None, kept=None, new_lengths=None, new_weights=None):
        """Keeps ``budget`` rows of each sequence and head (the first ``sinks``, the last ``recent``, and those of
        the largest ``weights``) and copies them in order to the pages of ``target_table``, in the same pools or in
        ``target_keys`` / ``target_values``.  The target pages must be others than the sequences' own.  Returns
        kept (int32 [batch, kv heads, budget] rows, -1 behind), the new lengths and the kept rows' weights
        (float32 [batch, kv heads, target rows], zeros behind)."""
        budget, sinks, recent = _count(budget, "budget"), _count(sinks, "sinks"), _count(recent, "recent")
        if (target_keys is None) != (target_values is None):
            raise ValueError("target_keys and target_values go together")
        if target_keys is None:
            target_keys, target_values = key_pages, value_pages
        if not (len(weights.shape) == 3 and len(key_pages.shape) == 4 and len(target_table.shape) == 2):
            raise ValueError("weights must be [batch, kv heads, rows], target_table [batch, pages], the pages 4-D")
        batch, heads = weights.shape[:2]
        if kept is None:
            kept = lengths.new_empty((batch, heads, budget))
        if new_lengths is None:
            new_lengths = lengths.new_empty(lengths.shape)
        if new_weights is None:
            new_weights = weights.new_empty((batch, heads, target_table.shape[1] * key_pages.shape[1]))
        invoke(arrays.EVICT, *self._where, key_pages, value_pages, page_table, lengths, weights, target_keys, target_values,
               target_table, kept, new_lengths, new_weights, budget, sinks, recent)
        return kept, new_lengths, new_weights

    # logits (include/miracle_cuda.h: mr_log_probabilities) ----------------------------
    def log_probabilities(self, logits, tokens=None, *, top=0, logprobs=None, entropy=None, top_tokens=None,
                          top_logprobs=None):
        """Of rows of ``logits`` [rows, vocabulary]: (logprobs, entropy, top_tokens, top_logprobs).  ``logprobs`` are
        the log probabilities of ``tokens`` (int32 [rows] or [rows, n]; one outside the vocabulary gives 0), None
        without them; ``entropy`` [rows] in nats; the ``top`` most likely tokens (at most 128) and their log
        probabilities [rows, top], falling, the lower token first where they are equal."""
        top = _count(top, "top")
        if len(getattr(logits, "shape", ())) != 2:
            raise ValueError("logits must be an array [rows, vocabulary]")
        rows = logits.shape[0]
        try:
            if tokens is not None and logprobs is None:
                logprobs = empty_like(logits, tokens.shape, "float32")
            if entropy is None:
                entropy = empty_like(logits, (rows,), "float32")
            if top_tokens is None:
                top_tokens = empty_like(logits, (rows, top), "int32")
            elif tuple(top_tokens.shape) != (rows, top):
                raise ValueError(f"top_tokens must be [{rows}, {top}]")
            if top_logprobs is None:
                top_logprobs = empty_like(logits, (rows, top), "float32")
        except AttributeError:   # found only here, so that arrays are not looked at twice
            for array, name, accessor in ((logits, "logits", "new_empty"), (tokens, "tokens", "shape"),
                                          (top_tokens, "top_tokens", "shape")):
                if array is not None and not hasattr(array, accessor):
                    raise _no_array(array, name) from None
            raise
        best = (top_tokens, top_logprobs) if top else (None, None)
        invoke(arrays.SCORE, *self._where, logits, tokens, logprobs, entropy, *best)
        return logprobs, entropy, top_tokens, top_logprobs

    def finish(self):
        call("mr_context_finish", self.context)
