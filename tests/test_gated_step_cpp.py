"""Runs the C++20 host layer's test of the step between two blocks and of 4-bit weights (tests/cpp/test_gated_step.cpp)."""
import os
import subprocess

import pytest


def _run(*args):
    from brodiffusion_amd import build
    if not os.path.exists(build.STEP_TEST):
        build.build_host()
    r = subprocess.run([build.STEP_TEST, *args], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "test_gated_step: OK" in r.stdout, r.stdout + r.stderr


def test_refusals_without_a_gpu():
    _run("--cpu")


@pytest.mark.gpu
def test_gated_step_executable():
    _run()
