"""How the library and its extension module are loaded, without a GPU."""

import os
import sys
import threading
import types
import warnings

import pytest
import torch

import llm_compileforge_b200 as package
from llm_compileforge_b200 import _lib, build, ops


@pytest.fixture
def unloaded(monkeypatch):
    _lib.load()  # (what is loaded once stays mapped; only the module's view of it is taken back)
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "calls", None)
    return monkeypatch


def test_a_second_thread_waits_until_the_calls_are_bound(unloaded):
    binding, go, seen = threading.Event(), threading.Event(), []
    bind = _lib._bind_calls

    def slow(lib):
        binding.set()
        assert go.wait(20)
        bind(lib)

    def use():
        _lib.load()
        seen.append(_lib.calls is not None)

    unloaded.setattr(_lib, "_bind_calls", slow)
    first, second = threading.Thread(target=use), threading.Thread(target=use)
    first.start()
    assert binding.wait(20)
    second.start()
    second.join(0.3)
    early = list(seen)
    go.set()
    first.join(20)
    second.join(20)
    assert early == [] and seen == [True, True]


def test_a_load_that_fails_is_tried_again(unloaded):
    def fails(lib):
        raise RuntimeError("bind")

    with unloaded.context() as m:
        m.setattr(_lib, "_bind_calls", fails)
        for _ in range(2):  # the second call is not answered with a library that is half set up
            with pytest.raises(RuntimeError, match="bind"):
                _lib.load()
    _lib.load()
    assert _lib.calls is not None


class Broken:
    """A finder for which the extension module is there but does not load."""

    def find_spec(self, name, path=None, target=None):
        if name.endswith("._calls"):
            raise ImportError("undefined symbol: _ZN3c10")


@pytest.fixture
def without_module(unloaded):
    unloaded.delattr(package, "_calls", raising=False)
    unloaded.delitem(sys.modules, package.__name__ + "._calls", raising=False)
    return unloaded


def bad_call_in_words():
    with pytest.raises(ValueError, match="K is zero"):
        ops.fused_linear(torch.zeros(4, 0), torch.zeros(0, 8))


def test_a_module_that_does_not_load_leaves_the_other_way(without_module):
    without_module.setattr(sys, "meta_path", [Broken(), *sys.meta_path])
    with pytest.warns(RuntimeWarning, match="undefined symbol.*build"):
        _lib.load()
    bad_call_in_words()


def test_a_module_that_is_not_built_leaves_the_other_way(without_module):
    class Absent(Broken):
        def find_spec(self, name, path=None, target=None):
            if name.endswith("._calls"):
                raise ModuleNotFoundError(name)

    without_module.setattr(sys, "meta_path", [Absent(), *sys.meta_path])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _lib.load()
    bad_call_in_words()


def test_a_module_of_another_torch_is_not_used(unloaded):
    unloaded.setattr(package, "_calls", types.SimpleNamespace(torch_version="1.0", bind=lambda *a: pytest.fail("bound")), raising=False)
    with pytest.warns(RuntimeWarning, match="1.0.*build"):
        _lib.load()
    bad_call_in_words()


def test_the_built_module_names_its_torch():
    from llm_compileforge_b200 import _calls

    assert _calls.torch_version == torch.__version__


@pytest.fixture
def calls_build(monkeypatch, tmp_path):
    """build.build_calls into an empty folder, the compiler replaced by one that notes its commands and writes its output."""
    commands = []

    def run(cmd):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")

    monkeypatch.setattr(build, "calls_path", lambda: str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    return lambda force=False: (build.build_calls(force, run), len(commands), os.path.exists(tmp_path / "_calls.so"))[1:]


def test_the_module_is_built_again_for_another_torch(calls_build, monkeypatch):
    assert calls_build() == (1, True) and calls_build() == (1, True)
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert calls_build() == (2, True) and calls_build() == (2, True)
    assert calls_build(force=True) == (3, True)


def test_without_torch_headers_the_library_is_built_all_the_same(calls_build, monkeypatch, tmp_path, capsys):
    from torch.utils import cpp_extension

    assert calls_build() == (1, True)
    monkeypatch.setattr(cpp_extension, "include_paths", lambda *a, **k: [str(tmp_path)])
    assert calls_build() == (1, True)  # still the one for this torch
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert calls_build() == (1, False)  # the one for another torch does not stay
    assert "headers" in capsys.readouterr().err


def test_without_a_compiler_no_module_older_than_its_sources_stays(calls_build, monkeypatch):
    assert calls_build() == (1, True)
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    assert calls_build() == (1, True)
    monkeypatch.setattr(build, "_headers_mtime", lambda: 1e12)  # the C ABI that it was built against is another now
    assert calls_build() == (1, False)


def test_without_torch_the_library_is_built_all_the_same(calls_build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert calls_build() == (0, False)
    assert "torch" in capsys.readouterr().err
