"""The C entry of gate_add_norm without a GPU: struct layout, and refusals ahead of any launch (what is passed as a tensor is never read); the kernels' instances."""
import ctypes as C
import os
import re
import subprocess

import pytest

from brodiffusion_amd import _capi as capi
from test_block_half_resources import TYPES, _wavefronts_and_chunks
from test_kernel_resources import kernels  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAR = 1 << 40


def test_struct_layout_matches_c(tmp_path):
    cls, name = capi.MiGateAddNormArgs, "mi_gate_add_norm_args"
    lines = [f'printf("%zu\\n", sizeof({name}));'] + [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mi_attention.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


# (4 rows of 64 columns: 512 bytes)
def _args(**kw):
    a = capi.MiGateAddNormArgs()
    a.struct_size, a.dtype, a.rows, a.cols, a.eps, a.post_eps, a.residual_scale = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 64, 1e-6, 1e-6, 1.0
    a.post_norm, a.norm = capi.MI_NORM_RMS, capi.MI_NORM_LAYER
    a.x, a.branch, a.gate, a.post_gain, a.gain, a.scale, a.shift, a.sum_out, a.out = (0x10000 * i for i in range(1, 10))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,said", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(cols=60), "multiple of 8"), (dict(cols=65544), "65536"), (dict(norm=3), "MI_NORM"),
    (dict(post_norm=-1), "MI_NORM"), (dict(eps=-1.0), "eps"), (dict(post_eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(residual_scale=float("inf")), "residual_scale"),
    (dict(residual_scale=float("nan")), "residual_scale"), (dict(x=None), "null"), (dict(out=None, sum_out=None), "neither"), (dict(out=None), "together"), (dict(norm=0), "together"),
    (dict(norm=0, out=None), "without a norm"), (dict(norm=0, out=None, gain=None, scale=None), "without a norm"), (dict(branch=None), "without a branch"),
    (dict(branch=None, gate=None, post_gain=None, post_norm=0), "without a branch"), (dict(post_norm=0), "without a post norm"), (dict(gate_rows=-1), "gate_rows"),
    (dict(scale_rows=-5), "scale_rows"), (dict(x_row_stride=60), "x must be a multiple"), (dict(x_row_stride=56), "x must be"), (dict(branch_row_stride=68), "branch"),
    (dict(gate_row_stride=60, gate_rows=1), "gate"), (dict(shift_row_stride=8, shift_rows=2), "shift"), (dict(out_row_stride=FAR + 8), "2^40"), (dict(scale_row_stride=FAR + 8, scale_rows=1), "2^40"),
    (dict(rows=0x7fffffff, x_row_stride=FAR), "2^56"), (dict(rows=0x7fffffff, gate_rows=1, gate_row_stride=FAR), "2^56"),
    (dict(x=0x10008), "x must be 16-byte"), (dict(gate=0x10008), "gate must be 16-byte"), (dict(gain=0x10008), "gain must be 16-byte"), (dict(out=0x10008), "out must be 16-byte"),
    (dict(out=0x10010), "out overlaps x"), (dict(sum_out=0x20010), "sum_out overlaps branch"), (dict(sum_out=0x90000), "out overlaps sum_out"), (dict(out=0x30070), "out overlaps gate"),
    (dict(sum_out=0x4fff0), "sum_out overlaps gain"), (dict(out=0x6fe10), "out overlaps shift"), (dict(out=0x30180, gate_rows=1), "out overlaps gate"), (dict(sum_out=0x60000), "overlaps scale"),
    (dict(out=0x40000), "overlaps post_gain")])
def test_refusals(fields, said):
    assert capi.lib().mi_gate_add_norm_forward(C.byref(_args(**fields))) == -1
    assert "mi_gate_add_norm_forward" in capi.last_error() and said in capi.last_error(), capi.last_error()


def test_no_rows_is_no_error():
    assert capi.lib().mi_gate_add_norm_forward(C.byref(_args(rows=0, x=None))) == 0


def test_kernels_are_those_that_calls_reach(kernels):
    reached = set()
    for rows in (1, 4096):
        for cols in range(8, 65537, 8):
            w, n = _wavefronts_and_chunks(rows, cols, 256)
            reached.add((w, {16: n if n in (2, 4, 8) else 4}.get(w, n)))
    for t in TYPES:
        built = {tuple(map(int, m.groups()[::-1])) for name in kernels if (m := re.search(rf"gate_norm_kernelI{t}Li(\d+)ELi(\d+)E", name))}
        assert built == reached


def test_no_scratch_memory(kernels):
    found = {name: (k[".private_segment_fixed_size"], k[".vgpr_spill_count"]) for name, k in kernels.items() if "gate_norm_kernelI" in name}
    assert found and not {name: use for name, use in found.items() if use != (0, 0)}
