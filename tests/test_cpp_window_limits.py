"""tests/cpp/test_window_limits.cpp: the windowed operators' C++ host side at the limits of what it is told."""
import importlib.util
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def _binary():
    spec = importlib.util.spec_from_file_location("build_cpp_tests", os.path.join(HERE, "cpp", "build_cpp_tests.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.SRC = os.path.join(HERE, "cpp", "test_window_limits.cpp")
    mod.OUT = os.path.join(mod.OUT_DIR, "test_window_limits")
    return mod.build()


def test_builds():
    assert os.path.exists(_binary())


@pytest.mark.gpu
def test_limits(cuda_device):
    res = subprocess.run([_binary()], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-4000:] + res.stderr[-2000:]
