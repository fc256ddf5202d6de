"""The Python extension for small calls of the 8-bit cache is an addition: neither the other libraries nor the operators depend on it."""
import sysconfig
import types
import warnings

import pytest
import torch

from kharon_b200 import _build, _native, ops

GPU = types.SimpleNamespace(is_cuda=True)


def test_the_other_libraries_are_built_without_it(monkeypatch, capsys, tmp_path):
    built = []
    monkeypatch.setattr(_build, "build_runtime", lambda force=False: built.append("rt") or tmp_path / "rt")
    monkeypatch.setattr(_build, "build_cuda", lambda force=False, verbose=False: built.append("cuda") or tmp_path / "cuda")

    def fails(force=False):
        built.append("bind")
        raise RuntimeError("build failed: no c10_cuda")
    monkeypatch.setattr(_build, "build_bind", fails)
    assert _build.build_all() == (tmp_path / "rt", tmp_path / "cuda")
    assert built == ["rt", "cuda", "bind"] and "no c10_cuda" in capsys.readouterr().err


def test_a_file_of_another_torch_or_python_is_not_loaded(monkeypatch):
    here = _build.bind_path()
    assert torch.__version__ in here.name and sysconfig.get_config_var("SOABI") in here.name
    monkeypatch.setattr(torch, "__version__", "9.8.7")
    assert _build.bind_path() != here and _build.bind_path().parent == here.parent
    monkeypatch.undo()
    monkeypatch.setattr(_native, "_bind", None)
    monkeypatch.setattr(_native, "cuda", lambda: None)
    asked = []

    def elsewhere():
        asked.append(1)
        return here.with_name("kharon_bind-of-another-torch.so")
    monkeypatch.setattr(_build, "bind_path", elsewhere)
    monkeypatch.setattr(_build, "build_bind", lambda force=False: pytest.fail("built") if not asked else (_ for _ in ()).throw(RuntimeError("no compiler")))
    with pytest.raises(RuntimeError, match="no compiler"):       # not there: built, not replaced by a file of another name
        _native.bind()


@pytest.mark.parametrize("error", [ImportError("undefined symbol"), OSError("no such file"), RuntimeError("build failed")])
def test_calls_go_through_ctypes_where_it_cannot_be_loaded(monkeypatch, error):
    tried = []

    def fails():
        tried.append(1)
        raise error
    monkeypatch.setattr(_native, "bind", fails)
    monkeypatch.setattr(ops, "_extension", None)
    monkeypatch.setattr(ops, "_lib", lambda: None)
    with pytest.warns(RuntimeWarning, match=str(error)):
        assert not ops._kv8_direct(GPU)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert not ops._kv8_direct(GPU) and len(tried) == 1      # said once, tried once


def test_a_missing_kernel_library_is_still_an_error(monkeypatch):
    def fails():
        raise RuntimeError("nvcc not found")
    monkeypatch.setattr(_native, "bind", fails)
    monkeypatch.setattr(ops, "_extension", None)
    monkeypatch.setattr(ops, "_lib", fails)
    with pytest.raises(RuntimeError, match="nvcc"):
        ops._kv8_direct(GPU)
    assert ops._extension is None
