"""Calls of the 8-bit rows and of the linear layer with an epilogue at the ends of what their documentation allows."""
import pytest
import torch

import brodiffusion_amd as bd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [64, 4104, 16392])
@pytest.mark.parametrize("power", [-62, -63, -64, -66, -68])
def test_norms_of_rows_whose_mean_square_is_no_normal_number(cols, power):
    """Without eps. A square of at least 2^-146 is off by at most half of FP32's fixed step 2^-149, as is each of the sums' roundings and the mean's:
    of values of 2^power (or twice that) the mean square is at least 2^(2 power), so that its relative error is at most (n + 2) 2^-150 / 2^(2 power) with
    n = 80 roundings in a row (64 terms of a lane and a tree), and half of that behind the root."""
    g = torch.Generator().manual_seed(cols)
    x = ((1 + torch.randint(0, 2, (3, cols), generator=g)) * (1 - 2 * torch.randint(0, 2, (3, cols), generator=g)) * 2.0 ** power).bfloat16().cuda()
    gain = (1 + 0.3 * torch.randn(cols, generator=g)).bfloat16().cuda()
    rel = (80 + 2) * 2.0 ** (-150 - 2 * power) / 2 + 46 * 2.0 ** -24
    z = x.double() * gain.double()
    inv = x.double().square().mean(dim=1).rsqrt()
    ref = z * inv[:, None]
    _, y = bd.add_rms_norm(x, None, gain, 0.0)
    _, q, scales = bd.add_rms_norm_int8(x, None, gain, 0.0)
    a = z.abs().amax(dim=1)
    assert torch.all((y.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + rel) * 1.01)
    assert torch.equal(q, torch.round(127 * z / a[:, None]).to(torch.int8))
    assert torch.all((scales.double() - a * inv / 127).abs() <= a * inv / 127 * rel * 1.01)
    if cols <= 16384:      # (the widest that this one takes)
        assert torch.equal(bd.rms_norm_rows(x, gain, 0.0), y)
