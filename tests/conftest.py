import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# Tests that hand invented addresses to a library call and count on its launch failing for want of a device.  Where a
# device is visible they run in a child process that sees none: such an address must never reach a GPU.
WITHOUT_DEVICES = {"test_shared_memory_is_refused_where_it_is_shared"}


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


def device_visible() -> bool:
    import torch

    return torch.cuda.is_available()


def run_without_devices(nodeid: str) -> subprocess.CompletedProcess:
    """One test in a process of its own that no CUDA device is visible to."""
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="")
    return subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", nodeid], capture_output=True, text=True, env=env, cwd=ROOT)


@pytest.hookimpl(tryfirst=True)
def pytest_pyfunc_call(pyfuncitem):
    if pyfuncitem.originalname not in WITHOUT_DEVICES or not device_visible():
        return None
    if os.environ.get("CUDA_VISIBLE_DEVICES") == "":
        pytest.fail("a CUDA device is visible in spite of CUDA_VISIBLE_DEVICES")
    path = os.path.relpath(str(pyfuncitem.path), ROOT)
    res = run_without_devices(f"{path}::{pyfuncitem.name}")
    if res.returncode:
        pytest.fail(res.stdout + res.stderr)
    return True


@pytest.fixture(scope="session")
def cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")
