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
