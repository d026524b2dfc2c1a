"""How the library and its extension module are loaded, without a GPU."""

import threading

import pytest

from llm_compileforge_b200 import _lib


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
