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


def test_the_binding_is_built_again_for_another_torch(build_native, tmp_path, monkeypatch):
    import torch

    commands = []

    class Done:
        returncode = 0

    def run(cmd, **kwargs):
        commands.append(cmd)
        build_native.BINDING_OUT.write_bytes(b"")
        return Done

    monkeypatch.setattr(build_native, "BINDING_OUT", tmp_path / "nb200_torch.so")
    monkeypatch.setattr(build_native, "OBJ_DIR", tmp_path)
    monkeypatch.setattr(build_native.subprocess, "run", run)
    for version, builds in ((torch.__version__, 1), (torch.__version__, 1), ("9.9.9+cu999", 2), ("9.9.9+cu999", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        build_native.build_binding()
        assert len(commands) == builds, version


def test_a_binding_of_another_torch_is_refused(native_lib, monkeypatch):
    import torch

    from neptune_mlir import native

    module = native.binding()
    assert module.torch_version == torch.__version__
    monkeypatch.setattr(native, "_BINDING", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    with pytest.raises(native.NativeLibraryError, match="built for torch .*, this is torch 9.9.9"):
        native.binding()
    assert native._BINDING is None


def test_a_binding_that_does_not_load_says_so(native_lib, tmp_path, monkeypatch):
    from neptune_mlir import native

    broken = tmp_path / "nb200_torch.so"
    broken.write_bytes(b"not a shared library")
    monkeypatch.setattr(native, "_BINDING", None)
    monkeypatch.setattr(native, "find_binding_path", lambda library=None: broken)
    with pytest.raises(native.NativeLibraryError, match="does not load"):
        native.binding()
