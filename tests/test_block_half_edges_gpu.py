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


# few rows, both sides of 8 features per compute unit; rings, parts, 256 x 256 tiles; rows too far apart for the rings
@pytest.mark.parametrize("M,N,K,stride", [(3, 64, 4096, 0), (9, 6144, 8192, 0), (40, 640, 2048, 0), (46, 368, 32000, 0), (600, 264, 1040, 0), (2188, 5392, 1024, 0),
                                          (40, 72, 1168, 8388608)])
def test_scales_of_rows_near_the_smallest_numbers(M, N, K, stride):
    """INT8 rows whose scales are no normal numbers and a result that is one: one rounding to bf16, 2^-8, and FP32 roundings of the sum, its product
    with a weight's scale and the fused rest, 3 2^-24. (Sums of at least K = 1024 positive products are above 2^20.)"""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x, w = (torch.randint(1, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((M, K), (N, K)))
    xs = (torch.randint(600, 1000, (M,), generator=g, device="cuda").double() * 2.0 ** -149).float()
    ws = (1 + torch.rand(N, generator=g, device="cuda")) / 16
    if stride:
        far = torch.zeros((M - 1) * stride + K, dtype=torch.int8, device="cuda").as_strided((M, K), (stride, 1))
        far.copy_(x)
        x = far
    y = bd.linear_act(x, w, x_scales=xs, w_scales=ws, dtype=torch.bfloat16)
    ref = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    assert bool((ref > 2.0 ** -125).all())
    assert torch.all((y.double() - ref).abs() <= ref * (2.0 ** -8 + 3 * 2.0 ** -24) * 1.001)


@pytest.mark.parametrize("kind", ["w16", "w8"])
@pytest.mark.parametrize("M", [3, 40, 300])
def test_activations_of_infinity(kind, M):
    """Sums of plus and minus infinity: x times what tends to 0 or 1, so infinity to the right and NaN to the left, in every activation."""
    x = torch.ones(M, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 5], x[1, 7], x[2, 9] = float("inf"), float("-inf"), float("nan")
    w = torch.ones(72, 64, device="cuda", dtype=torch.int8 if kind == "w8" else torch.bfloat16)
    for act in ("gelu", "gelu_tanh", "silu"):
        y = bd.linear_act(x, w, activation=act, w_scales=torch.ones(72, device="cuda") if kind == "w8" else None)
        assert bool((y[0] == float("inf")).all()) and torch.isnan(y[1:3]).all() and torch.isfinite(y[3:]).all(), act
