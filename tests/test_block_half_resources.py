"""What the built library says of the kernels of the 8-bit rows and of the linear layer with an epilogue: no scratch memory, and no instance that no call
reaches. tests/test_kernel_resources.py reads the metadata."""
import re

import pytest

from test_kernel_resources import kernels  # noqa: F401

TYPES = ("DF16_", "DF16b")


@pytest.mark.parametrize("kernel,at_least", [("rows_kernel", 2), ("linear_few_kernel", 2), ("linear_join_kernel", 2), ("linear_kernel", 2), ("linear_pipe_kernel", 2), ("linear_dma_kernel", 2)])
def test_no_scratch_memory(kernels, kernel, at_least):
    found = {name: (k[".private_segment_fixed_size"], k[".vgpr_spill_count"]) for name, k in kernels.items() if re.search(r"\d" + kernel + "I", name)}
    assert len(found) >= at_least
    assert not {name: use for name, use in found.items() if use != (0, 0)}


def _wavefronts_and_chunks(rows, cols, compute_units):
    """What the rule of rows_int8.hip, as its comment has it, gives a row"""
    chunks, each = (cols + 7) // 8, 3 if rows >= 4 * compute_units else 2
    for w, most in ((1, 64 * each), (2, 128 * each), (4, 256 * each), (8, 2048 if each == 3 else 1024), (16, 8192)):
        if chunks <= most:
            n = -(-chunks // (64 * w))
            return w, (n if n <= 4 else 8)


def test_rows_kernels_are_those_that_calls_reach(kernels):
    reached = {_wavefronts_and_chunks(rows, cols, 256) for rows in (1, 4096) for cols in range(8, 65537, 8)}
    for t in TYPES:
        for norm in (0, 1):
            built = {tuple(map(int, m.groups()[::-1])) for name in kernels if (m := re.search(rf"rows_kernelI{t}Li(\d+)ELi(\d+)ELb{norm}E", name))}
            assert built == reached
