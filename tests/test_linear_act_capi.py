"""The C entries of the 8-bit rows and of the linear layer with an epilogue, without a GPU: struct layouts, and refusals ahead of any launch (what
is passed as a tensor is never read)."""
import ctypes as C
import os
import subprocess

import pytest

from brodiffusion_amd import _capi as capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_c(tmp_path):
    pairs = [("mi_add_rms_norm_args", capi.MiAddRmsNormArgs), ("mi_quantize_rows_args", capi.MiQuantizeRowsArgs), ("mi_linear_act_args", capi.MiLinearActArgs)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mi_attention.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def _norm(**kw):
    a = capi.MiAddRmsNormArgs()
    a.struct_size, a.dtype, a.rows, a.cols, a.eps = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 64, 1e-6
    a.x, a.residual, a.gain, a.sum_out, a.out = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _rows(**kw):
    a = capi.MiQuantizeRowsArgs()
    a.struct_size, a.dtype, a.rows, a.cols = C.sizeof(a), capi.MI_DTYPE_F16, 4, 64
    a.x, a.out_q, a.out_scales = 0x10000, 0x20000, 0x30000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _linear(**kw):
    a = capi.MiLinearActArgs()
    a.struct_size, a.dtype, a.rows, a.in_features, a.out_features = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 64, 40
    a.x, a.w, a.bias, a.residual, a.y = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


REFUSED = [
    ("mi_add_rms_norm_forward", _norm, [
        (dict(struct_size=8), "struct_size"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(cols=60), "multiple of 8"), (dict(cols=0), "multiple of 8"),
        (dict(cols=65544), "65536"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(out=None), "neither"), (dict(out_q=0x60000), "together"),
        (dict(out_scales=0x60000), "together"), (dict(residual=None), "without a residual"), (dict(x=None), "null"), (dict(gain=None), "null"),
        (dict(gain=0x30008), "gain must be"), (dict(x=0x10008), "x must be 16-byte"), (dict(x_row_stride=56), "row stride of x"), (dict(out_row_stride=68), "row stride of out"),
        (dict(sum_out=0x50000), "out overlaps sum_out"), (dict(out=0x10010), "out overlaps x"), (dict(sum_out=0x20080), "sum_out overlaps residual"),
        (dict(out_q=0x10000, out_scales=0x60000), "out_q overlaps x"), (dict(out_q=0x60000, out_scales=0x60040), "out_scales overlaps out_q"),
        (dict(out_q=0x60004, out_scales=0x70000), "8-byte aligned"), (dict(out_q=0x60000, out_scales=0x70002), "4-byte"),
        (dict(out_q=0x60000, out_scales=0x70000, q_row_stride=60), "row stride of out_q"), (dict(out=0x30000), "out overlaps gain"),
        (dict(sum_out=0x2ff80), "sum_out overlaps gain"), (dict(out_q=0x60000, out_scales=0x30010), "out_scales overlaps gain"),
        (dict(x_row_stride=1 << 41), "exceeds 2^40")]),
    ("mi_quantize_rows_forward", _rows, [
        (dict(struct_size=8), "struct_size"), (dict(dtype=0), "dtype"), (dict(cols=4), "multiple of 8"), (dict(x=None), "null"), (dict(out_q=None), "null"),
        (dict(out_scales=None), "null"), (dict(out_q=0x10040), "overlaps"), (dict(x_row_stride=60), "row stride")]),
    ("mi_linear_act_forward", _linear, [
        (dict(struct_size=8), "struct_size"), (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(in_features=60), "multiple of 8"), (dict(out_features=36), "of 8"),
        (dict(in_features=0), "features"), (dict(activation=4), "activation"), (dict(activation=-1), "activation"), (dict(x_scales=0x60000), "INT8 weights"),
        (dict(x_scales=0x60000, w_scales=0x70000, in_features=72), "multiple of 16"), (dict(x_scales=0x60000, w_scales=0x70000, in_features=131072), "131056"),
        (dict(x_scales=0x60000, w_scales=0x70000, x_row_stride=72), "row strides"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
        (dict(x_row_stride=60), "row strides"), (dict(x_row_stride=56), "smaller"), (dict(residual_row_stride=32), "smaller"), (dict(bias=0x30008), "16-byte"),
        (dict(w_scales=0x60002), "4-byte"), (dict(y=0x40010), "overlaps the residual"), (dict(y=0x40000, y_row_stride=48), "overlaps the residual"),
        (dict(y=0x10020), "overlaps x"), (dict(y=0x20100), "overlaps w"), (dict(y=0x10100, x_row_stride=96, residual=None), "overlaps x"),
        (dict(y=0x30010), "overlaps the bias"), (dict(y=0x5ff00, w_scales=0x60000), "overlaps scales"),
        (dict(y=0x50000, x_scales=0x50004, w_scales=0x70000), "overlaps scales"), (dict(in_features=(1 << 30) + 8), "2^30"),
        (dict(rows=(1 << 30) + 1), "2^30"), (dict(out_features=(1 << 30) + 8), "2^30"), (dict(w_row_stride=1 << 41), "exceeds 2^40")]),
]


@pytest.mark.parametrize("entry,make,fields,text", [(e, m, f, t) for e, m, cases in REFUSED for f, t in cases])
def test_refused_calls(entry, make, fields, text):
    fn = getattr(capi.lib(), entry)
    assert fn(C.byref(make(**fields))) == -1
    assert entry in capi.last_error() and text in capi.last_error()


def test_null_args_and_no_rows():
    for entry, make in (("mi_add_rms_norm_forward", _norm), ("mi_quantize_rows_forward", _rows), ("mi_linear_act_forward", _linear)):
        fn = getattr(capi.lib(), entry)
        assert fn(None) == -1 and "null args" in capi.last_error()
        assert fn(C.byref(make(rows=0, x=None))) == 0


def test_tensors_on_the_cpu_are_refused():
    import torch

    import brodiffusion_amd as bd
    x, g = torch.zeros(2, 64, dtype=torch.half), torch.ones(64, dtype=torch.half)
    for call in (lambda: bd.add_rms_norm(x, x, g, 1e-6), lambda: bd.add_rms_norm_int8(x, None, g, 1e-6), lambda: bd.quantize_rows_int8(x),
                 lambda: bd.linear_act(x, torch.zeros(8, 64, dtype=torch.half))):
        with pytest.raises(RuntimeError, match="not on the GPU"):
            call()
