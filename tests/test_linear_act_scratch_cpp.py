"""Runs the C++20 host layer's test of the scratch behind linear layers (tests/cpp/test_linear_act_scratch.cpp)."""
import os
import subprocess

import pytest

from brodiffusion_amd import build


def test_the_executable_is_built():
    if not os.path.exists(build.SCRATCH_TEST):
        build.build_host()
    assert os.access(build.SCRATCH_TEST, os.X_OK)


@pytest.mark.gpu
def test_scratch_grows_and_stays():
    if not os.path.exists(build.SCRATCH_TEST):
        build.build_host()
    r = subprocess.run([build.SCRATCH_TEST], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "test_linear_act_scratch: OK" in r.stdout, r.stdout + r.stderr
