"""perf/operators.py's calls of the framework go to the stream and the device that torch works on at that moment."""
import importlib.util
import sys
from types import SimpleNamespace

import pytest

from conftest import PACKAGE, REPO


@pytest.fixture
def measured():
    spec = importlib.util.spec_from_file_location("measured_operators", REPO / "perf" / "operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_backend_for_each_stream_and_device(measured, monkeypatch):
    made = []

    def backend(device_index=0, stream=None):
        made.append((device_index, stream))
        return SimpleNamespace(device_index=device_index, stream=stream)

    now = SimpleNamespace(device_index=0, cuda_stream=11)
    monkeypatch.setitem(sys.modules, PACKAGE, SimpleNamespace(CUDABackend=backend))
    monkeypatch.setattr(measured.torch.cuda, "current_stream", lambda *a: now)
    monkeypatch.setattr(measured.torch.accelerator, "current_stream", lambda *a: (now.device_index, now.cuda_stream))
    first = measured._backend()
    assert (first.device_index, first.stream) == (0, 11)
    now = SimpleNamespace(device_index=0, cuda_stream=12)
    assert measured._backend().stream == 12
    now = SimpleNamespace(device_index=1, cuda_stream=12)
    assert (measured._backend().device_index, measured._backend().stream) == (1, 12)
    now = SimpleNamespace(device_index=0, cuda_stream=11)
    assert measured._backend() is first and len(made) == 3


@pytest.mark.gpu
def test_a_case_on_a_side_stream(measured):
    import torch
    measured.own = True
    case = dict(op="paged", type="bf16", batch=3, heads=8, kv_heads=2, dim=64, length=700, page=16, window=0, sinks=0,
                spread=1, weights=True)
    want = [x.clone() for x in measured.run(measured.prepare(case, 5))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = measured.run(measured.prepare(case, 5))
    side.synchronize()   # the side stream alone: the work was queued on it
    assert all(torch.equal(x, y) for x, y in zip(got, want))
