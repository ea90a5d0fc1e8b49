"""Arrays described through DLPack's exchange in C, and those that only look as if they offered it: the same bytes as by
the accessors."""
import pytest

from conftest import submodule
from test_array_calls import Stub


class NoCapsule(Stub):
    __dlpack_c_exchange_api__ = 17


def capsule(name, table):
    import ctypes
    new = ctypes.pythonapi.PyCapsule_New
    new.restype, new.argtypes = ctypes.py_object, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
    return new(ctypes.addressof(table), name, None)


def offering(name, major, answer):
    """A type whose exchange is of a version and returns an answer, and what has to outlive it."""
    import ctypes
    entry = ctypes.PYFUNCTYPE(ctypes.c_int, ctypes.py_object, ctypes.c_void_p)(lambda array, to: answer)
    table = (ctypes.c_uint64 * 7)(major, 0, 0, 0, 0, ctypes.cast(entry, ctypes.c_void_p).value, 0)
    kept = table, entry, name
    return type("Offering", (Stub,), {"__dlpack_c_exchange_api__": capsule(name, table), "kept": kept})


@pytest.mark.parametrize("make", [lambda: Stub, lambda: NoCapsule, lambda: type("Heir", (NoCapsule,), {}),
                                  lambda: offering(b"another", 1, 0), lambda: offering(b"dlpack_exchange_api", 2, 0),
                                  lambda: offering(b"dlpack_exchange_api", 1, -1)])
def test_other_types_are_read_by_their_accessors(make):
    arrays, kind = submodule("arrays"), make()
    for _ in range(3):
        assert arrays.describe(kind(), "x", 0) == arrays.described(kind(), "x", 0)
        with pytest.raises(ValueError, match="x"):
            arrays.describe(kind(), "x", 1)


def test_host_tensors_are_refused():
    import torch
    arrays = submodule("arrays")
    with pytest.raises(ValueError):
        arrays.describe(torch.zeros(4), "x", 0)


@pytest.mark.gpu
def test_tensors_of_all_kinds():
    import torch
    arrays = submodule("arrays")
    x = torch.zeros(6, 5, 4, 8, device="cuda")
    parameter = torch.nn.Parameter(torch.zeros(3, 3, device="cuda"))
    made = [x, x[1:, 2:4], x.permute(2, 0, 3, 1), x[:0], x[:, :1, 0], x[0, 0, 0], x[:1].expand(7, -1, -1, -1), parameter,
            torch.zeros(2, 2, device="cuda", requires_grad=True)]
    made += [torch.ones(3, 4, device="cuda").to(t)[1:, ::2] for t in (torch.float16, torch.bfloat16, torch.int32, torch.uint8)]
    for t in made:
        assert arrays.describe(t, "x", 0) == arrays.described(t, "x", 0)
    for t in (torch.zeros(3, device="cuda", dtype=torch.bool), torch.zeros(3, device="cuda", dtype=torch.float64),
              torch.zeros(3, device="cuda", dtype=torch.int8), torch.zeros((), device="cuda"), x[None]):
        with pytest.raises(ValueError):
            arrays.describe(t, "x", 0)
