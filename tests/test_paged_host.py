"""The paged cache's operators without a GPU: what they refuse, before any device work, and array descriptions."""
import ctypes as C
import struct

import numpy as np
import pytest

from conftest import submodule

F32, F16, BF16, I32 = range(4)


class Fake:
    """An array's description without memory behind it: nothing is read before a call is refused."""

    def __init__(self, shape, dtype=BF16, stride=None, pointer=1 << 20):
        self.shape, self.code, self.pointer = tuple(shape), dtype, pointer
        self.strides = tuple(stride) if stride else tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def packed(self):
        n, pad = len(self.shape), (0,) * (4 - len(self.shape))
        return struct.pack("<Qii8q", self.pointer, self.code, n, *self.shape, *pad, *self.strides, *pad)


def refused(name, arrays, *scalars):
    lib = submodule("_native").library()
    code = getattr(lib, name)(None, *[x.packed() if x is not None else None for x in arrays], *scalars)
    assert code == 1   # MR_ERR_ARGUMENT
    return lib.mr_last_error().decode()


def pools(**kw):
    return Fake((10, 16, 4, 64), **kw), Fake((10, 16, 4, 64), pointer=1 << 24, **kw)


def paged(**changes):
    k, v = pools()
    args = dict(query=Fake((3, 8, 64)), key_pages=k, value_pages=v, table=Fake((3, 5), I32), lengths=Fake((3,), I32),
                weights=None, out=Fake((3, 8, 64), pointer=1 << 28), window=0, sinks=0, scale=0.125)
    args.update(changes)
    values = list(args.values())
    return refused("mr_paged_attention", values[:7], *values[7:])


def test_valid_arguments_reach_the_context():
    # with nothing wrong, the missing context is what is left to refuse
    assert paged() == "ctx is NULL"
    assert paged(weights=Fake((3, 4, 80), F32)) == "ctx is NULL"


@pytest.mark.parametrize("changes, message", [
    (dict(query=Fake((3, 6, 64)), out=Fake((3, 6, 64), pointer=1 << 28)), "multiple of the pages' 4 heads"),
    (dict(query=Fake((3, 8, 32)), out=Fake((3, 8, 32), pointer=1 << 28)), "32 values a head, the pages 64"),
    (dict(query=Fake((3, 8, 64), F16)), "of one type"),
    (dict(query=Fake((3, 8))), "must have 3 dimensions"),
    (dict(query=None), "query is missing"),
    (dict(query=Fake((3, 8, 64), pointer=(1 << 20) + 8)), "16-byte boundary"),
    (dict(query=Fake((3, 8, 64), stride=(516, 64, 1))), "stride 0 is not a multiple of 16 bytes"),
    (dict(query=Fake((3, 8, 64), stride=(1024, 128, 2))), "last dimension must be contiguous"),
    (dict(query=Fake((3, 8, 64), stride=(-512, 64, 1))), "stride 0 is out of range"),
    (dict(query=Fake((3, 8, 64), pointer=0)), "no memory"),
    (dict(out=Fake((3, 8, 64))), "must not share memory"),
    (dict(out=Fake((3, 8, 64), stride=(0, 64, 1), pointer=1 << 28)), "must not overlap itself"),
    (dict(out=Fake((2, 8, 64), pointer=1 << 28)), "differ in shape"),
    (dict(lengths=Fake((2,), I32)), "lengths must have 3 values"),
    (dict(lengths=Fake((3,), F32)), "lengths must be int32"),
    (dict(table=Fake((2, 5), I32)), "a row for each of the 3 sequences"),
    (dict(table=Fake((3, 1 << 27), I32)), "too many rows"),
    (dict(weights=Fake((3, 4, 79), F32)), "weights must be \\[3, 4, 80\\]"),
    (dict(weights=Fake((3, 4, 80), BF16)), "weights must be float32"),
    (dict(window=-1), "must not be negative"),
    (dict(sinks=-1), "must not be negative"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(value_pages=Fake((10, 16, 4, 64), F16)), "of one floating type"),
    (dict(value_pages=Fake((9, 16, 4, 64))), "differ in shape"),
    (dict(key_pages=Fake((10, 16, 4, 64), stride=(1 << 32, 256, 64, 1))), "stride 0 passes 4 GB"),
    (dict(key_pages=Fake((10, 16, 4, 64), stride=(1 << 60, 256, 64, 1))), "stride 0 is out of range"),
    (dict(key_pages=Fake((10, 16, 4, 60)), value_pages=Fake((10, 16, 4, 60))), "whole 16-byte pieces"),
    (dict(key_pages=Fake((10, 16, 4, 136)), value_pages=Fake((10, 16, 4, 136))), "at most 128 values"),
])
def test_paged_attention_refuses(changes, message):
    import re
    assert re.search(message, paged(**changes))


def window(**changes):
    args = dict(query=Fake((50, 8, 64)), keys=Fake((90, 4, 64)), values=Fake((90, 4, 64)), qo=Fake((4,), I32),
                ko=Fake((4,), I32), out=Fake((50, 8, 64), pointer=1 << 28), window=0, sinks=0, scale=0.125)
    args.update(changes)
    values = list(args.values())
    return refused("mr_window_attention", values[:6], *values[6:])


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(ko=Fake((3,), I32)), "one value more"),
    (dict(qo=Fake((0,), I32), ko=Fake((0,), I32)), "one value more"),
    (dict(keys=Fake((90, 3, 64)), values=Fake((90, 3, 64))), "multiple of the 3 key heads"),
    (dict(values=Fake((91, 4, 64))), "keys and values differ"),
    (dict(values=Fake((90, 4, 64), F32)), "one floating type"),
    (dict(query=Fake((50, 8, 64), I32)), "one floating type"),
    (dict(keys=Fake((90, 4, 128)), values=Fake((90, 4, 128))), "64 values a head, keys 128"),
    (dict(out=Fake((50, 8, 64))), "must not share memory"),
    (dict(qo=Fake((4,), F32)), "must be int32"),
    (dict(scale=float("inf")), "scale must be finite"),
])
def test_window_attention_refuses(changes, message):
    assert message in window(**changes)


def append(**changes):
    k, v = pools()
    args = dict(keys=Fake((7, 4, 64)), values=Fake((7, 4, 64)), key_pages=k, value_pages=v, table=Fake((3, 5), I32),
                lengths=Fake((3,), I32), offsets=Fake((4,), I32))
    args.update(changes)
    return refused("mr_append_pages", list(args.values()))


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(offsets=None), "one row for each of the 3 sequences"),
    (dict(offsets=Fake((3,), I32)), "offsets must have 4 values"),
    (dict(keys=Fake((7, 4, 64), F32)), "of one type"),
    (dict(keys=Fake((7, 2, 64)), values=Fake((7, 2, 64))), "as the pages' heads and dim"),
    (dict(values=Fake((6, 4, 64))), "keys and values differ"),
    (dict(key_pages=Fake((10, 16, 4, 64), stride=(0, 256, 64, 1))), "must not overlap itself"),
])
def test_append_pages_refuses(changes, message):
    assert message in append(**changes)


def evict(**changes):
    k, v = pools()
    args = dict(key_pages=k, value_pages=v, table=Fake((3, 5), I32), lengths=Fake((3,), I32),
                weights=Fake((3, 4, 80), F32), target_keys=k, target_values=v, target=Fake((3, 2), I32),
                kept=Fake((3, 4, 20), I32), new_lengths=Fake((3,), I32, pointer=1 << 21),
                new_weights=Fake((3, 4, 32), F32, pointer=1 << 22), budget=20, sinks=2, recent=4)
    args.update(changes)
    values = list(args.values())
    return refused("mr_evict_pages", values[:11], *values[11:])


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(budget=5), "budget 5 is less than sinks 2 and recent 4"),
    (dict(budget=0), "budget must be positive"),
    (dict(recent=-1), "not negative"),
    (dict(target=Fake((3, 1), I32), new_weights=Fake((3, 4, 16), F32, pointer=1 << 22)), "room for 16 rows of the 20"),
    (dict(kept=Fake((3, 4, 19), I32)), "kept must be \\[3, 4, 20\\]"),
    (dict(new_weights=Fake((3, 4, 32), F32)), "must not share memory"),
    (dict(new_lengths=Fake((3,), I32)), "must not share memory"),
    (dict(target_keys=Fake((10, 8, 4, 64)), target_values=Fake((10, 8, 4, 64))), "the pages' rows, heads and dim"),
    (dict(target_keys=Fake((10, 16, 4, 64), F16), target_values=Fake((10, 16, 4, 64), F16)), "the pages' type"),
    (dict(weights=Fake((3, 4, 64), F32)), "weights must be \\[3, 4, 80\\]"),
])
def test_evict_pages_refuses(changes, message):
    import re
    assert re.search(message, evict(**changes))


def test_a_full_context_needs_room_for_what_it_holds():
    # a budget above the table's rows keeps all of them: room for those is enough
    assert evict(budget=500, kept=Fake((3, 4, 500), I32), target=Fake((3, 5), I32),
                 new_weights=Fake((3, 4, 80), F32, pointer=1 << 22)) == "ctx is NULL"


class Stub:
    """What describe() asks of an array."""

    def __init__(self, shape, dtype="float32", device=0):
        self.shape, self.dtype, self.device = shape, dtype, device

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def data_ptr(self):
        return 4096

    def get_device(self):
        return self.device


def test_descriptions():
    import torch
    arrays = submodule("arrays")
    got = arrays.describe(Stub((2, 3, 4), "bfloat16"), "x", 0)
    assert struct.unpack("<Qii8q", got) == (4096, BF16, 3, 2, 3, 4, 0, 12, 4, 1, 0)
    assert struct.unpack("<Qii8q", arrays.describe(Stub((5,), torch.int32), "x", 0))[1] == I32
    for bad, message in ((Stub((2,), "float64"), "unsupported array type"), (Stub((2,), device=1), "on device 0, not 1"),
                         (Stub((2,), device=-1), "not the host"), (Stub(()), "1 to 4 dimensions"),
                         (Stub((1, 1, 1, 1, 1)), "1 to 4 dimensions"), (np.zeros(3), "not ndarray"),
                         (torch.zeros(3), "not the host")):
        with pytest.raises(ValueError, match=message):
            arrays.describe(bad, "x", 0)


def test_host_values_of_bfloat16_arrays():
    arrays = submodule("arrays")
    values = np.array([1.0, -2.5, 3.1415927, 1e-20], np.float32)
    raw = arrays.stored(values, "bfloat16")
    assert raw.dtype == np.uint16 and arrays.host_type("bfloat16") == np.uint16
    assert np.all(np.abs(arrays.widened(raw, "bfloat16") - values) <= 2.0 ** -8 * np.abs(values))
    assert C.sizeof(C.c_int64) * 8 + 16 == len(arrays.describe(Stub((1,)), "x", 0))
