"""The refusals of the C++ host layer of rows and heads (anode_b200/host/anode_rows.hpp), on any machine: tests/cpp/test_host_rows_refusals.cpp."""
import os
import subprocess

import pytest

from tests.test_cpp_host import CPP, build


@pytest.mark.parametrize("which", ["missing", "shapes"])
def test_refused_before_anything_is_asked_of_a_device(which):
    build()
    r = subprocess.run([os.path.join(CPP, "test_host_rows_refusals"), which], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failed" in r.stdout, (r.returncode, r.stdout, r.stderr)
