"""The C++ host side of the operators around windowed attention: tests/cpp/test_window.cpp is built as
the other C++ tests are; without a GPU only its refusals run."""
import importlib.util
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def _binary():
    spec = importlib.util.spec_from_file_location("build_cpp_tests", os.path.join(HERE, "cpp", "build_cpp_tests.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.SRC = os.path.join(HERE, "cpp", "test_window.cpp")
    mod.OUT = os.path.join(mod.OUT_DIR, "test_window")
    return mod.build()


def test_builds_and_refuses():
    res = subprocess.run([_binary(), "--check"], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.mark.gpu
def test_a_step_matches_plain_loops(cuda_device):
    res = subprocess.run([_binary()], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-4000:] + res.stderr[-2000:]
