"""More refusals of the C entries of the 8-bit rows and of the linear layer with an epilogue, ahead of any launch (nothing passed as a tensor is read)."""
import ctypes as C

import pytest

from brodiffusion_amd import _capi as capi
from test_linear_act_capi import _linear, _norm, _rows

FAR = 1 << 40      # the largest row stride


@pytest.mark.parametrize("entry,make,fields", [
    ("mi_linear_act_forward", _linear, dict(rows=1 << 30, x_row_stride=FAR)),
    ("mi_linear_act_forward", _linear, dict(rows=1 << 30, y_row_stride=FAR)),
    ("mi_linear_act_forward", _linear, dict(rows=1 << 30, residual_row_stride=FAR, x_row_stride=64)),
    ("mi_linear_act_forward", _linear, dict(out_features=1 << 30, w_row_stride=FAR)),
    ("mi_linear_act_forward", _linear, dict(rows=(1 << 22) + 2, x_row_stride=1 << 34)),
    ("mi_add_rms_norm_forward", _norm, dict(rows=0x7fffffff, x_row_stride=FAR)),
    ("mi_add_rms_norm_forward", _norm, dict(rows=0x7fffffff, out_row_stride=FAR)),
    ("mi_add_rms_norm_forward", _norm, dict(rows=0x7fffffff, residual_row_stride=FAR, sum_row_stride=FAR)),
    ("mi_quantize_rows_forward", _rows, dict(rows=0x7fffffff, x_row_stride=FAR)),
    ("mi_quantize_rows_forward", _rows, dict(rows=0x7fffffff, q_row_stride=FAR)),
])
def test_rows_that_reach_past_any_address(entry, make, fields):
    """Rows times stride beyond 2^56 elements: what would not fit the 64-bit offsets of the checks for overlaps."""
    assert getattr(capi.lib(), entry)(C.byref(make(**fields))) == -1
    assert entry in capi.last_error() and "reach over more than 2^56 elements" in capi.last_error()


def test_rows_that_reach_just_so_far_are_not_refused_for_it():
    a = _linear(rows=(1 << 16) + 1, x_row_stride=FAR, y=0x10100, residual=None)      # (and the overlap is found)
    assert capi.lib().mi_linear_act_forward(C.byref(a)) == -1 and "overlaps x" in capi.last_error()
    a = _norm(rows=(1 << 16) + 1, x_row_stride=FAR, sum_out=0x10010)
    assert capi.lib().mi_add_rms_norm_forward(C.byref(a)) == -1 and "sum_out overlaps x" in capi.last_error()


# (64 features of 4 rows: x 512 bytes, w 40 x 128, bias 80, residual and y 320)
@pytest.mark.parametrize("kind", ["w16", "w8", "w8a8"])
@pytest.mark.parametrize("name,at", [("x", 0x10000), ("x", 0x100f0), ("w", 0x20000), ("w", 0x209f0), ("bias", 0x30040), ("residual", 0x40130), ("y", 0x50000), ("y", 0x50130)])
def test_scratch_that_is_part_of_an_operand(kind, name, at):
    more = {"w16": {}, "w8": dict(w_scales=0x60000), "w8a8": dict(w_scales=0x60000, x_scales=0x70000)}[kind]
    for scratch, size in ((at, 64), (at - 0x400, 0x410)):
        a = _linear(scratch=scratch, scratch_bytes=size, **more)
        assert capi.lib().mi_linear_act_forward(C.byref(a)) == -1
        assert f"scratch overlaps {name}" in capi.last_error(), capi.last_error()


def test_scratch_that_is_part_of_the_scales():
    for fields, name in ((dict(scratch=0x60080), "w_scales"), (dict(scratch=0x70000, scratch_bytes=1 << 47), "x_scales"), (dict(scratch=0x6ff00, scratch_bytes=0x110), "x_scales")):
        a = _linear(w_scales=0x60000, x_scales=0x70000, **{"scratch_bytes": 64, **fields})
        assert capi.lib().mi_linear_act_forward(C.byref(a)) == -1
        assert f"scratch overlaps {name}" in capi.last_error()


def test_what_would_be_used_does_not_hang_on_the_scratch_fields():
    a = _linear(scratch=0x10000, scratch_bytes=1 << 20, rows=46, in_features=15984, out_features=368, x=0x1000000, w=0x2000000, y=0x4000000, residual=None)
    need = capi.lib().mi_linear_act_scratch_bytes(C.byref(a))
    a.scratch, a.scratch_bytes = 0x2000000, 1 << 20
    assert need > 0 and capi.lib().mi_linear_act_scratch_bytes(C.byref(a)) == need
