"""What the built library says of the kernels of the 8-bit rows and of the linear layer with an epilogue: no scratch memory. tests/test_kernel_resources.py reads the metadata."""
import re

import pytest

from test_kernel_resources import kernels  # noqa: F401

@pytest.mark.parametrize("kernel,at_least", [("rows_kernel", 2), ("linear_few_kernel", 2), ("linear_join_kernel", 2), ("linear_kernel", 2), ("linear_pipe_kernel", 2), ("linear_dma_kernel", 2)])
def test_no_scratch_memory(kernels, kernel, at_least):
    found = {name: (k[".private_segment_fixed_size"], k[".vgpr_spill_count"]) for name, k in kernels.items() if re.search(r"\d" + kernel + "I", name)}
    assert len(found) >= at_least
    assert not {name: use for name, use in found.items() if use != (0, 0)}
