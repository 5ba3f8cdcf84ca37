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
