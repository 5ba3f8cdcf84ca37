"""The C entries of the linear layer with 4-bit weights without a GPU: struct layouts, sizes, and refusals ahead of any launch (what is passed as a tensor is never read)."""
import ctypes as C
import os
import subprocess

import pytest

from brodiffusion_amd import _capi as capi
from test_kernel_resources import kernels  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAR = 1 << 40


def test_struct_layouts_match_c(tmp_path):
    pairs = [("mi_pack_int4_args", capi.MiPackInt4Args), ("mi_linear_int4_args", capi.MiLinearInt4Args)]
    lines, want = [], []
    for name, cls in pairs:
        lines += [f'printf("%zu\\n", sizeof({name}));'] + [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mi_attention.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    assert [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()] == want


@pytest.mark.parametrize("n,k,size", [(8, 8, 1024), (16, 128, 1024), (24, 136, 4096), (16384, 6144, 16384 * 6144 // 2), (0, 128, 0), (16, -8, 0), (1 << 30, 1 << 30, 1 << 59)])
def test_packed_bytes(n, k, size):
    assert capi.lib().mi_int4_packed_bytes(n, k) == size


# (4 rows, 264 in, 40 out, groups of 64: x 2112 bytes, w 9216, scales 400, zeros 200, bias 80, residual and y 320)
def _linear(**kw):
    a = capi.MiLinearInt4Args()
    a.struct_size, a.dtype, a.rows, a.in_features, a.out_features, a.group = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 264, 40, 64
    a.x, a.w, a.scales, a.zeros, a.bias, a.residual, a.y = (0x10000 * i for i in range(1, 8))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _pack(**kw):
    a = capi.MiPackInt4Args()
    a.struct_size, a.out_features, a.in_features = C.sizeof(a), 40, 264
    a.q, a.packed = 0x10000, 0x20000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,said", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(in_features=0), "features"), (dict(out_features=-8), "features"),
    (dict(in_features=260), "multiples of 8"), (dict(out_features=36), "multiples of 8"), (dict(in_features=(1 << 30) + 8), "2^30"), (dict(activation=4), "activation"), (dict(activation=-1), "activation"),
    (dict(group=0), "group"), (dict(group=-64), "group"), (dict(group=16), "group"), (dict(group=96), "group"), (dict(group=192), "group"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(scales=None), "null"), (dict(y=None), "null"), (dict(x_row_stride=268), "multiples"), (dict(x_row_stride=256), "smaller"), (dict(y_row_stride=32), "smaller"), (dict(residual_row_stride=8), "smaller"),
    (dict(y_row_stride=FAR + 8), "2^40"), (dict(rows=1 << 30, x_row_stride=FAR), "2^56"), (dict(x=0x10008), "16-byte"), (dict(scales=0x30008), "16-byte"), (dict(bias=0x50002), "16-byte"), (dict(zeros=0x40004), "8-byte"),
    (dict(y=0x60010), "overlaps the residual"), (dict(y=0x60000, y_row_stride=48), "overlaps the residual"), (dict(y=0x10100, residual=None), "overlaps x"), (dict(y=0x223f0), "overlaps w"),
    (dict(y=0x30180), "overlaps scales"), (dict(y=0x3fed0), "overlaps zeros"), (dict(y=0x4fed0), "overlaps the bias")])
def test_refusals(fields, said):
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(**fields))) == -1
    assert "mi_linear_int4_forward" in capi.last_error() and said in capi.last_error(), capi.last_error()


@pytest.mark.parametrize("fields,said", [
    (dict(struct_size=8), "struct_size"), (dict(in_features=260), "multiples of 8"), (dict(out_features=0), "features"), (dict(q=None), "null"), (dict(packed=None), "null"), (dict(q_row_stride=128), "stride"),
    (dict(q_row_stride=134), "stride"), (dict(q_row_stride=FAR + 4), "2^56"), (dict(out_features=1 << 30, q_row_stride=1 << 34), "2^56"), (dict(q=0x10002), "4-byte"), (dict(packed=0x20008), "16-byte"),
    (dict(packed=0x11490), "overlaps"), (dict(q=0x223fc), "overlaps")])
def test_pack_refusals(fields, said):
    assert capi.lib().mi_pack_int4(C.byref(_pack(**fields))) == -1
    assert "mi_pack_int4" in capi.last_error() and said in capi.last_error(), capi.last_error()


def test_no_rows_is_no_error():
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(rows=0, x=None))) == 0
