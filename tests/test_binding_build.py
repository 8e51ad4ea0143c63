"""Building and loading the torch binding, without a GPU."""

import importlib.util
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "mlir-toy_b200"


@pytest.fixture
def build_native(native_lib):
    spec = importlib.util.spec_from_file_location("nb200_build_native_under_test", PKG / "build_native.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_kernel_library_is_built_without_the_binding(build_native, monkeypatch):
    """No torch, or one without the libraries to link with: the C ABI and the operators that use it alone are still there."""
    def no_torch(force=False):
        raise RuntimeError("g++ failed on torch_binding.cpp: cannot find -lc10_cuda")

    monkeypatch.setattr(build_native, "build_binding", no_torch)
    with pytest.warns(RuntimeWarning, match="cannot find -lc10_cuda"):
        assert build_native.build() == build_native.OUT
    assert build_native.OUT.exists()
