"""Runs the C++20 host layer's test of the 8-bit rows and the linear layer with an epilogue (tests/cpp/test_block_half.cpp)."""
import os
import subprocess

import pytest


def _run(*args):
    from brodiffusion_amd import build
    if not os.path.exists(build.BLOCK_TEST):
        build.build_host()
    r = subprocess.run([build.BLOCK_TEST, *args], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "test_block_half: OK" in r.stdout, r.stdout + r.stderr


def test_refusals_without_a_gpu():
    _run("--cpu")


@pytest.mark.gpu
def test_block_half_executable():
    _run()
