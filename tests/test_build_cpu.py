"""The build's stamps: what makes libnv4.so and its torch binding stale, and the
library without the binding (no compiler runs here)."""
import importlib.util
import os
import sysconfig

import pytest
import torch

from nanovllm import _native

PACKAGE = os.path.dirname(os.path.dirname(os.path.abspath(_native.__file__)))


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """The build script, writing to a folder of its own through a compiler that makes empty files."""
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(PACKAGE, "build_native.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.OUT_DIR = str(tmp_path)
    mod.OUT, mod.BINDING = (str(tmp_path / n) for n in ("libnv4.so", "_nv4_serving.so"))
    mod.built = []

    def run(cmd, failure):
        target = cmd[cmd.index("-o") + 1]
        mod.built.append(os.path.basename(target)[:-len(".tmp")])
        open(target, "w").close()
        return ""
    monkeypatch.setattr(mod, "_run", run)
    return mod


def test_nothing_is_built_twice(builder):
    assert builder.build() == builder.OUT
    assert builder.built == ["libnv4.so", "_nv4_serving.so"]
    builder.build()
    assert len(builder.built) == 2
    builder.build(force=True)
    assert len(builder.built) == 4


@pytest.mark.parametrize("what", ["torch", "python", "abi"])
def test_another_torch_or_python_makes_the_binding_stale(builder, monkeypatch, what):
    builder.build()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    elif what == "abi":
        monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: False)
    else:
        inner = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda n: ".other.so" if n == "EXT_SUFFIX" else inner(n))
    del builder.built[:]
    builder.build()
    assert builder.built == ["_nv4_serving.so"]
    builder.build()
    assert builder.built == ["_nv4_serving.so"]


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    path = os.path.join(os.path.dirname(_native.LIB_PATH), "_nv4_serving.so")
    _native._check_fresh(path, "binding_hash")
    _native.load()
    monkeypatch.setattr(_native, "_serving", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(_native.NativeLibraryError, match="rebuild"):
        _native.serving()


def test_the_library_alone(builder, monkeypatch):
    """Neither torch nor a host compiler's module is needed for the C ABI."""
    def no_torch():
        raise ImportError("torch")
    monkeypatch.setattr(builder, "binding_hash", no_torch)
    monkeypatch.setattr(builder, "_binding_command", no_torch)
    builder.build(binding=False)
    assert builder.built == ["libnv4.so"]
    with pytest.raises(ImportError):
        builder.build()
    builder.build(binding=False)  # the library stays current
    assert builder.built == ["libnv4.so"]


def test_a_failed_build_leaves_no_stamp(builder, monkeypatch):
    builder.build()

    def fail(cmd, failure):
        raise RuntimeError(failure)
    monkeypatch.setattr(builder, "_run", fail)
    with pytest.raises(RuntimeError, match="nvcc"):
        builder.build(force=True)
    assert not os.path.exists(builder.OUT + ".srchash") and os.path.exists(builder.BINDING + ".srchash")
