"""linear_act on rows too far apart for 32-bit offsets within a tile: few rows, and what the rings leave to the tiles through registers: x's and w's, on both sizes
(128 x 128 from two tiles per compute unit on). tests/test_linear_act_gpu.py derives the bounds."""
import pytest
import torch

import brodiffusion_amd as bd
from test_linear_act_gpu import call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", ["w16", "w8", "w8a8"])
@pytest.mark.parametrize("M,N,K,far", [(33, 65544, 80, "x"), (65537, 72, 80, "w"), (40, 136, 144, "w"), (70, 72, 208, "xw"), (20, 72, 208, "xw")])
def test_far_rows(kind, dtype, M, N, K, far):
    large = -(-M // 128) * -(-N // 128) >= 2 * bd.device_info()["compute_units"]
    assert large == (M * N > 1_000_000)
    c = make(M + N, kind, M, N, K, dtype)
    for name in far:
        t = c[name]
        stride = 4_194_304 * (2 if kind == "w8a8" else 1) + 16
        # (what lies between the rows is never read: 127 or NaN there would show)
        buf = torch.full(((t.shape[0] - 1) * stride + K,), 127 if t.dtype == torch.int8 else float("nan"), dtype=t.dtype, device="cuda")
        c[name] = buf.as_strided((t.shape[0], K), (stride, 1))
        c[name].copy_(t)
    wide = torch.full((M + 1, N + 8), 7.0, dtype=c["dt"], device="cuda")
    act = {"w16": "gelu", "w8": "silu", "w8a8": "gelu_tanh"}[kind]
    call(c, act, out=wide[:M, :N])
    check(c, act, wide[:M, :N], far)
    assert bool((wide[M:] == 7).all()) and bool((wide[:, N:] == 7).all())
    assert call(c, act, out=c["residual"]) is c["residual"] and torch.equal(c["residual"], wide[:M, :N])
