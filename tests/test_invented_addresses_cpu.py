"""Calls on invented addresses never run where a CUDA device is visible."""

import ast
import os
import subprocess

import pytest

import conftest

TESTS = os.path.dirname(os.path.abspath(__file__))
NAME = "test_shared_memory_is_refused_where_it_is_shared"


class Item:
    """What the hook asks of a test item."""

    def __init__(self, name):
        self.name = self.originalname = name
        self.path = os.path.join(TESTS, "test_feed_forward_cpu.py")


def test_the_tests_that_count_on_a_failing_launch_are_known():
    found = set()
    for f in os.listdir(TESTS):
        if f.startswith("test_") and f.endswith(".py") and f != os.path.basename(__file__):
            with open(os.path.join(TESTS, f)) as fh:
                text = fh.read()
            found |= {d.name for d in ast.walk(ast.parse(text))
                      if isinstance(d, ast.FunctionDef) and d.name.startswith("test_") and "fails at the launch" in ast.get_source_segment(text, d)}
    assert found == {NAME} == conftest.WITHOUT_DEVICES


def test_they_run_in_a_child_without_devices(monkeypatch):
    seen = []

    def run(cmd, env, **kw):
        seen.append((cmd, env["CUDA_VISIBLE_DEVICES"]))
        return subprocess.CompletedProcess(cmd, len(seen) - 1, "", "")

    monkeypatch.delenv("CUDA_VISIBLE_DEVICES", raising=False)
    monkeypatch.setattr(conftest, "device_visible", lambda: True)
    monkeypatch.setattr(conftest.subprocess, "run", run)
    assert conftest.pytest_pyfunc_call(Item(NAME)) is True  # done: pytest does not call the function here
    assert seen[0][0][-1] == f"tests/test_feed_forward_cpu.py::{NAME}" and seen[0][1] == ""
    with pytest.raises(pytest.fail.Exception):  # the child failed
        conftest.pytest_pyfunc_call(Item(NAME))
    assert conftest.pytest_pyfunc_call(Item("test_names_of_the_executor")) is None  # every other test runs as always
    monkeypatch.setenv("CUDA_VISIBLE_DEVICES", "")  # a child that sees a device all the same refuses
    with pytest.raises(pytest.fail.Exception, match="visible"):
        conftest.pytest_pyfunc_call(Item(NAME))
    assert len(seen) == 2
    monkeypatch.setattr(conftest, "device_visible", lambda: False)
    assert conftest.pytest_pyfunc_call(Item(NAME)) is None


def test_the_child_sees_no_device_and_passes():
    res = conftest.run_without_devices(f"tests/test_feed_forward_cpu.py::{NAME}")
    assert res.returncode == 0, res.stdout + res.stderr
