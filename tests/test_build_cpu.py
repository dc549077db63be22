"""CPU: the torch binding is built and loaded for the Python and torch at hand only, and who has not what it needs can still build the library."""

import importlib.util
import os
import subprocess
import sys
import sysconfig

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def builder():
    spec = importlib.util.spec_from_file_location("feather_b200_build", os.path.join(ROOT, "comfyui-featherops_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_a_binding_of_another_torch_or_python_is_not_loaded(native, monkeypatch):
    loaded = []
    real = importlib.machinery.ExtensionFileLoader
    monkeypatch.setattr(native.importlib.machinery, "ExtensionFileLoader", lambda *a: loaded.append(a) or real(*a))
    for owner, name, value in ((torch, "__version__", "0.1.0+cu1"), (native.importlib.machinery, "EXTENSION_SUFFIXES", [".cpython-31-none.so"])):
        with monkeypatch.context() as m:
            m.setattr(native, "_binding", None)
            m.setattr(owner, name, value)
            with pytest.raises(native.FeatherNativeError, match="build.py"):
                native.binding()
    assert not loaded
    assert native.binding() is not None


def test_the_builder_and_the_loader_mean_the_same_file(builder, native):
    assert builder.binding_path() == native.binding_path()
    assert torch.__version__ in os.path.basename(builder.binding_path()) and builder.binding_path().endswith(sysconfig.get_config_var("EXT_SUFFIX"))


@pytest.mark.parametrize("missing", ["headers of Python", "headers of torch", "compiler", "torch"])
def test_the_library_builds_without_what_the_binding_needs(builder, monkeypatch, tmp_path, capsys, missing):
    assert builder.binding_unavailable() is None
    if missing == "headers of Python":
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    elif missing == "headers of torch":
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    elif missing == "compiler":
        monkeypatch.setattr(builder.shutil, "which", lambda name: None if name in ("c++", "g++") else "/usr/local/cuda/bin/" + name)
    else:
        monkeypatch.setitem(sys.modules, "torch", None)
    assert missing in builder.binding_unavailable()
    monkeypatch.setattr(builder, "build_library", lambda **kw: "the library")
    assert builder.build_all(force=True) == ["the library"]
    assert missing in capsys.readouterr().err


def test_a_binding_that_does_not_compile_is_an_error(builder, monkeypatch, tmp_path):
    bad = tmp_path / "binding.cpp"
    bad.write_text("#error no\n")
    monkeypatch.setattr(builder, "BINDING_SRC", str(bad))
    monkeypatch.setattr(builder, "binding_path", lambda: str(tmp_path / "out.so"))
    with pytest.raises(RuntimeError, match="failed to build"):
        builder.build_binding(force=True)


def test_the_script_prints_what_it_built():
    res = subprocess.run([sys.executable, os.path.join(ROOT, "comfyui-featherops_b200", "build.py")], stdout=subprocess.PIPE, text=True, check=True)
    assert [os.path.exists(line) for line in res.stdout.split()] == [True, True]
