"""Runs the C++ test of the token layers (tests/cpp/test_tokens.cpp) on the GPU, in a process of its own."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "build", "test_tokens")


def test_cpp_tokens():
    assert os.path.exists(EXE), f"{EXE} is missing: run `make -C tests/cpp`"
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=110)
    print(r.stdout[-2000:], r.stderr[-2000:])
    assert r.returncode == 0, f"exit status {r.returncode}\n" + r.stdout[-2000:] + r.stderr[-2000:]
