"""Normalization over rows and rotary positions in the C++ host layer (anode_b200/host/anode_rows.hpp): builds the test program of tests/cpp
and, on a GPU, runs it.  Without a GPU it must link, load the library and report that it found no device."""
import os
import subprocess

import pytest

from tests.test_cpp_host import CPP, build

BIN = os.path.join(CPP, "test_host_rows")


def test_cpp_rows_build_and_load():
    build()
    import torch
    if torch.cuda.is_available():
        pytest.skip("covered by the GPU test")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "no CUDA device" in r.stderr, (r.returncode, r.stdout, r.stderr)


@pytest.mark.gpu
def test_cpp_rows_on_gpu():
    build()
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "0 tests failed" in r.stdout, r.stdout + r.stderr
