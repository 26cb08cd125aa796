"""CPU tests of the build script: the C library does not depend on the PyTorch binding."""

import ctypes
import importlib.util
import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def script(tmp_path, monkeypatch):
    """The build script on a library of one function, in a folder of its own."""
    spec = importlib.util.spec_from_file_location("gtk_build_script", os.path.join(REPO, "genie-tk_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "one.cpp").write_text('extern "C" __attribute__((visibility("default"))) int one(void) { return 41; }\n')
    monkeypatch.setattr(mod, "CSRC", str(csrc))
    monkeypatch.setattr(mod, "BUILD", str(tmp_path / "objects"))
    monkeypatch.setattr(mod, "OUT", str(tmp_path / "lib" / "libone.so"))
    monkeypatch.setattr(mod, "BINDING_OUT", str(tmp_path / "lib" / "_gtk_torch.so"))
    return mod


def test_without_pytorch_the_c_library_is_built(script, monkeypatch, capfd):
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch fails
    assert script.build() == script.OUT
    assert ctypes.CDLL(script.OUT).one() == 41
    assert not os.path.exists(script.BINDING_OUT)
    assert "PyTorch" in capfd.readouterr().err


def test_a_binding_that_does_not_compile_fails_behind_the_library(script, monkeypatch, tmp_path):
    bad = tmp_path / "binding.cpp"
    bad.write_text("#error no binding\n")
    monkeypatch.setattr(script, "BINDING_SRC", str(bad))
    with pytest.raises(RuntimeError, match="no binding"):
        script.build()
    assert ctypes.CDLL(script.OUT).one() == 41
    assert not os.path.exists(script.BINDING_OUT)
