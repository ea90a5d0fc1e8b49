"""The C module of the array operators' calls: needed by those alone, built for one interpreter."""
from pathlib import Path

from conftest import submodule


class Stub:
    """What describe() asks of an array."""

    shape, dtype = (1,), "float32"

    def stride(self):
        return (1,)

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 0


def test_the_package_without_its_built_modules(tmp_path):
    """Models, backends and errors can be named where nothing is built, or _pycall for another interpreter only; the
    array operators alone need it, and say so."""
    import shutil
    import subprocess
    import sys
    package = Path(submodule("arrays").__file__).parent
    shutil.copytree(package, tmp_path / package.name, ignore=shutil.ignore_patterns("*.so", "_build", "csrc", "__pycache__"))
    (tmp_path / package.name / "_pycall.so").write_text("another's")
    (tmp_path / package.name / "_pycall.cpython-27.so").write_text("another's")
    run = subprocess.run([sys.executable, "-c", f"""
import importlib
pkg = importlib.import_module({package.name!r})
assert pkg.MiracleModel and pkg.CUDABackend and pkg.Tensor and pkg.ModelConfig
arrays = importlib.import_module({package.name!r} + ".arrays")
for call in (lambda: arrays.describe(None, "x", 0), lambda: arrays._pycall()):
    try:
        call()
    except pkg.CUDAError as error:
        assert str(arrays.PYCALL) in str(error) and "build.py" in str(error)
    else:
        raise AssertionError("described without _pycall")
print("named")
"""], cwd=tmp_path, capture_output=True, text=True, timeout=120)
    assert run.stdout.strip() == "named", run.stderr


def test_the_module_is_built_for_this_interpreter():
    import sysconfig
    arrays, build = submodule("arrays"), submodule("build")
    assert arrays.PYCALL == build.PYCALL and arrays.PYCALL.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    arrays.describe(Stub(), "x", 0)
    assert Path(arrays._pycall().__file__) == arrays.PYCALL
