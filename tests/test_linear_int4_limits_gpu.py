"""linear_int4 at the ends of what it takes, on every kind of kernel: groups far longer than the contraction, the largest finite rows."""
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


@pytest.mark.parametrize("m,k", [(1, 264), (40, 264), (200, 520), (2049, 264), (1, 8200), (200, 8200)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, True), (128, True), (128, False)])
def test_the_largest_rows(m, k, group, zeros):
    """bf16 values up to 2^112 with any zero point: (15 + 255) 128 2^112 is below 2^128, so no partial sum ahead of the scale overflows, and the bounds hold as they do elsewhere"""
    g = torch.Generator().manual_seed(m + k + group)
    n, t = 264, torch.bfloat16
    q, scales, z = _checkpoint(g, n, k, group, zeros, t)
    scales = (scales.float() * 2.0 ** -110).to(t)
    if zeros:
        z = torch.randint(0, 256, z.shape, generator=g, dtype=torch.uint8).cuda()
    x = ((2 * torch.rand(m, k, generator=g) - 1) * 2.0 ** 112).to(t).cuda()
    x[0, :128] = 2.0 ** 112      # (all of one sign: the largest sum that there is)
    y = bd.linear_int4(x, bd.pack_int4(q, scales, z, group=group))
    _check(y, *_reference(x, q, scales, z, group, None, "none", None))
