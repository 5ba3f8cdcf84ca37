"""The C entries of the linear layer with 4-bit weights at the ends of what they take, without a GPU: refusals ahead of any launch (what is passed as a tensor is never read)."""
import ctypes as C

import pytest

from brodiffusion_amd import _capi as capi

MOST_GROUP = 0x7fffff80      # the largest multiple of 128 that a C int holds


# (4 rows, 264 in, 40 out: scales and zeros of one group are 80 and 40 bytes)
def _linear(**kw):
    a = capi.MiLinearInt4Args()
    a.struct_size, a.dtype, a.rows, a.in_features, a.out_features, a.group = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 264, 40, 128
    a.x, a.w, a.scales, a.zeros, a.y = 0x10000, 0x20000, 0x30000, 0x40000, 0x70000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,said", [(dict(y=0x30040), "y overlaps scales"), (dict(y=0x40020), "y overlaps zeros"), (dict(scratch=0x30040, scratch_bytes=64), "scratch overlaps scales")])
@pytest.mark.parametrize("group", [384, 1 << 30, MOST_GROUP])
def test_the_longest_groups_are_one(group, fields, said):
    """in_features + group - 1 past a C int came out as no group at all, and the one before the first was read"""
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(group=group, **fields))) == -1
    assert said in capi.last_error(), capi.last_error()


# work-items of a grid's first dimension, by the form's index (csrc/linear_int4_forms.h): 512 for each run of features, 256 for each tile of eight at a time
ROWS_FEATURES = ((16, 16), (16, 32), (16, 64), (32, 64), (32, 128), (64, 128), (64, 192), (96, 192), (64, 256))


def _across(form, m, n):
    r, f = ROWS_FEATURES[form]
    return -(-n // f) * 512 if form < 3 else -(-(-(-m // r) * -(-n // f)) // 8) * 8 * 256


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n", [(1 << 30, 8), (1 << 30, 264), (1 << 27, 1160), (1 << 24, 8200), (1 << 30, 1 << 14), (1, 1 << 25), (5000, 1 << 25), (1, (1 << 27) + 8), (1, 1 << 28), (1, (1 << 29) - 8), (1, 1 << 29),
                                 (16, 1 << 30), (1 << 20, 1 << 24), (1 << 30, 1 << 30)])
def test_grids_that_hold(group, m, n):
    """Fewer than 2^32 work-items across; where no form has so few the call is refused, not handed to a launch that fails"""
    import os
    from brodiffusion_amd import build
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    shares = C.c_int()
    form = C.CDLL(build.FORMS_LIB).int4_form_test(m, n, 8, C.c_long(8), group, 256, C.c_ulong(0), C.byref(shares))
    fits = [f for f in range(9) if _across(f, m, n) < 1 << 32 and not (f < 3 and m > 65535 * 16) and not (f >= 3 and n > 1 << 24) and (group, f) not in ((32, 2), (32, 8), (64, 8))]
    assert form in fits if fits else form < 0
    if not fits:
        far = 1 << 50      # (addresses that no operand reaches from another)
        a = _linear(rows=m, in_features=8, out_features=n, group=group, x=far, w=2 * far, scales=3 * far, zeros=None, y=4 * far)
        assert capi.lib().mi_linear_int4_forward(C.byref(a)) == -1
        assert ("rows reach over" if m * n > 1 << 56 else "problem too large for one launch") in capi.last_error(), capi.last_error()
        assert capi.lib().mi_linear_int4_scratch_bytes(C.byref(a)) == 0
