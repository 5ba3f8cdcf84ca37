"""Runs the C++20 host layer's test of pack_int4's sizes (tests/cpp/test_int4_sizes.cpp); it needs no GPU."""
import os
import subprocess


def test_int4_sizes_executable():
    from brodiffusion_amd import build
    if not os.path.exists(build.SIZES_TEST):
        build.build_host()
    r = subprocess.run([build.SIZES_TEST], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "test_int4_sizes: OK" in r.stdout, r.stdout + r.stderr
