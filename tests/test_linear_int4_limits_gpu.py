"""linear_int4 at the ends of what it takes, on every kind of kernel: groups far longer than the contraction."""
import dataclasses

import pytest
import torch

import brodiffusion_amd as bd
from test_linear_int4_gpu import _check, _checkpoint, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 40, 200, 2049])
@pytest.mark.parametrize("k", [264, 8200])
def test_groups_longer_than_the_contraction(m, k):
    """One group, whatever its nominal length: up to the largest multiple of 128 that a C int holds"""
    g = torch.Generator().manual_seed(m + k)
    n = 264
    q, scales, z = _checkpoint(g, n, k, 1 << 20, True, torch.bfloat16)
    w = bd.pack_int4(q, scales, z, group=-(-k // 128) * 128)
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    want = bd.linear_int4(x, w)
    _check(want, *_reference(x, q, scales, z, w.group, None, "none", None))
    for group in (1 << 30, 0x7fffff80):
        assert torch.equal(bd.linear_int4(x, bd.pack_int4(q, scales, z, group=group)), want)
        assert torch.equal(bd.linear_int4(x, dataclasses.replace(w, group=group)), want)
