"""add_rms_norm, add_rms_norm_int8 and quantize_rows_int8 against their definitions in 64 bits: widths of one chunk, one past a wavefront's, one
past a work group's and the largest; rows that are zero, tiny, huge or not finite; ties; strides; outputs that are their inputs.

The stored sum is one rounding of an FP32 addition, so it is compared bit for bit, and the integers are defined as exactly rounded quotients, so
they are too. Scales: a product, a quotient, and the reciprocal root (2 units) of a sum of n squares in FP32, whose relative error is at most
(n + 2) 2^-24 at any order and half of that behind the root; the kernels add at most 64 terms in a row, then in a tree, so n here is 80.
16-bit outputs: the same and half a step of the type, eps / 2."""
import numpy as np
import pytest
import torch

import brodiffusion_amd as bd
from helpers import TORCH_DT

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
REL = (80 / 2 + 2 + 4) * EPS32       # of inv, with the few roundings around it
SIZES = [(1, 8), (3, 64), (5, 512), (4, 520), (7, 1160), (333, 2240), (2, 2568), (9, 3080), (2, 4096), (3, 4104), (1, 6144), (5, 10248), (2, 16384), (3, 16392),
         (2, 33000), (1, 65536), (1031, 1152)]


def _make(seed, rows, cols, dtype):
    g = torch.Generator().manual_seed(seed)
    loud = torch.exp(torch.randn(cols, generator=g))
    x, r = ((torch.randn(rows, cols, generator=g) * loud).to(TORCH_DT[dtype]).cuda() for _ in range(2))
    gain = (1 + 0.3 * torch.randn(cols, generator=g)).to(TORCH_DT[dtype]).cuda()
    return x, r, gain


def _steps(z):
    """Rows of FP32 values to the integers: 127 z / a in 64 bits is no tie unless the quotient is one (both sides have under 32 bits)."""
    a = z.abs().amax(dim=1, keepdim=True).double()
    return torch.round(127.0 * z.double() / torch.where(a > 0, a, torch.ones_like(a))).to(torch.int8), a.squeeze(1)


def _inv(h, eps):
    return (h.double().square().mean(dim=1) + eps).rsqrt()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("with_residual", [True, False], ids=["residual", "plain"])
def test_norm_rows(dtype, rows, cols, with_residual):
    x, r, gain = _make(7 * rows + cols, rows, cols, dtype)
    res, eps, half = (r if with_residual else None), 1e-5, torch.finfo(TORCH_DT[dtype]).eps / 2
    h = (x.float() + r.float()).to(x.dtype) if with_residual else x
    inv = _inv(h, eps)
    s16, y = bd.add_rms_norm(x, res, gain, eps)
    s8, q, scales = bd.add_rms_norm_int8(x, res, gain, eps)
    assert torch.equal(s16, h) and torch.equal(s8, h)
    if not with_residual:
        assert s16 is x and s8 is x
    ref = h.double() * gain.double() * inv[:, None]
    # (below the smallest normal number of the type a step is a fixed one)
    assert torch.all((y.double() - ref).abs() <= ref.abs() * (half + REL) + torch.finfo(y.dtype).tiny * half)
    want, a = _steps(h.float() * gain.float())
    assert q.dtype == torch.int8 and torch.equal(q, want)
    ref = a * inv / 127
    assert scales.shape == (rows,) and torch.all((scales.double() - ref).abs() <= ref * REL)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize_rows(dtype, rows, cols):
    x, _, _ = _make(11 * rows + cols, rows, cols, dtype)
    q, scales = bd.quantize_rows_int8(x)
    want, a = _steps(x.float())
    assert torch.equal(q, want)
    assert torch.all((scales.double() - a / 127).abs() <= a / 127 * 2 * EPS32)


def test_quantize_ties_go_to_the_even_integer():
    """a = 127 makes every half a tie: 0.5 -> 0, 1.5 -> 2, 2.5 -> 2, ... of both signs, at three scales."""
    half = torch.arange(0, 127, dtype=torch.float32) + 0.5
    row = torch.cat([half, -half, torch.tensor([127.0, -127.0])])
    x = torch.stack([row, row * 2.0 ** -20, row * 2.0 ** 6]).bfloat16().cuda()
    assert torch.equal(x[0].float().cpu(), row)      # 8 bits are enough for these
    q, _ = bd.quantize_rows_int8(x)
    want = torch.round(row).to(torch.int8)      # to even
    for i in range(3):
        assert torch.equal(q[i].cpu(), want)


def test_quantize_next_to_ties():
    """fp16 rows of every value of one binade below their maximum, for maxima of 11 bits: quotients as near to a tie as the type gives."""
    for a in (1025.0, 1365.0, 1777.0, 2047.0):
        v = torch.arange(0, 2048, dtype=torch.float32)
        v = v[v <= a]
        x = torch.zeros(1, 2048)
        x[0, :len(v)] = v
        x[0, 0] = -a
        q, _ = bd.quantize_rows_int8(x.half().cuda())
        assert torch.equal(q.cpu(), _steps(x)[0])


@pytest.mark.parametrize("magnitude", [2.0 ** -130, 2.0 ** -100, 2.0 ** -61, 1.0, 2.0 ** 60, 2.0 ** 125])
def test_quantize_tiny_and_huge_rows(magnitude):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(6, 1032, generator=g).clamp(-3, 3) * magnitude).bfloat16().cuda()
    q, scales = bd.quantize_rows_int8(x)
    want, a = _steps(x.float())
    assert torch.equal(q, want)
    # (a scale below 2^-126 has fixed steps of 2^-149)
    assert torch.all((scales.double() - a / 127).abs() <= a / 127 * 2 * EPS32 + 2.0 ** -149)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("cols", [72, 4104])
def test_rows_of_zeros_and_rows_that_are_not_finite(dtype, cols):
    x, r, gain = _make(5, 9, cols, dtype)
    r[:] = 0
    x[1] = 0
    x[3, 17], x[4, 70], x[6, 0], x[6, 5] = float("nan"), float("inf"), float("-inf"), float("inf")
    fine = torch.tensor([True, True, True, False, False, True, False, True, True], device="cuda")
    ones = torch.ones_like(gain)
    for q, scales, z in ((*bd.quantize_rows_int8(x), x.float()), (*bd.add_rms_norm_int8(x, r, gain, 1e-6)[1:], x.float() * gain.float()),
                         (*bd.add_rms_norm_int8(x, None, ones, 1e-6)[1:], x.float())):
        assert torch.equal(torch.isnan(scales), ~fine) and scales[1] == 0 and bool((q[~fine] == 0).all()) and bool((q[1] == 0).all())
        assert torch.equal(q[fine], _steps(z[fine])[0])
    h, y = bd.add_rms_norm(x, r, gain, 1e-6)
    assert torch.equal(torch.isnan(h), torch.isnan(x)) and torch.equal(torch.isinf(h), torch.isinf(x))
    assert torch.isfinite(y[fine]).all() and bool((y[1] == 0).all())
    assert torch.isnan(y[3]).all() and all(torch.isnan(y[i, c]) for i, c in ((4, 70), (6, 0), (6, 5)))


def test_rows_that_are_zero_without_eps():
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    gain = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    _, q, scales = bd.add_rms_norm_int8(x, None, gain, 0.0)
    assert bool((q == 0).all()) and bool((scales == 0).all())


@pytest.mark.parametrize("cols", [328, 4616, 17000])
def test_outputs_that_are_inputs_and_strides(cols):
    """Every tensor a column slice of a wider one; the sum into X or the residual, the norm into either; what lies beside the slices stays."""
    x0, r0, gain = _make(19, 13, cols, "bf16")
    h = (x0.float() + r0.float()).to(x0.dtype)
    want_h, want_y = bd.add_rms_norm(x0, r0, gain, 1e-6)
    _, want_q, want_s = bd.add_rms_norm_int8(x0, r0, gain, 1e-6)
    assert torch.equal(want_h, h)

    def wide(t, pad):
        w = torch.full((t.shape[0], t.shape[1] + 2 * pad), 3, dtype=t.dtype, device="cuda")
        w[:, pad:-pad] = t
        return w, w[:, pad:-pad]

    for into in ("x", "residual", "both", "swapped"):
        (xw, x), (rw, r) = wide(x0, 8), wide(r0, 16)
        s_out, y_out = {"x": (x, None), "residual": (r, None), "both": (x, r), "swapped": (r, x)}[into]
        s, y = bd.add_rms_norm(x, r, gain, 1e-6, sum_out=s_out, out=y_out)
        assert s is s_out and torch.equal(s, want_h) and torch.equal(y, want_y)
        for w, pad in ((xw, 8), (rw, 16)):
            assert bool((w[:, :pad] == 3).all()) and bool((w[:, -pad:] == 3).all())
        if into != "both":
            continue
        (xw, x), (rw, r) = wide(x0, 8), wide(r0, 16)
        qw, q = wide(torch.zeros(13, cols, dtype=torch.int8, device="cuda"), 24)
        s, q2, sc = bd.add_rms_norm_int8(x, r, gain, 1e-6, sum_out=r, out=q)
        assert s is r and q2 is q and torch.equal(q, want_q) and torch.equal(sc, want_s) and torch.equal(r, want_h) and torch.equal(x, x0)
        assert bool((qw[:, :24] == 3).all()) and bool((qw[:, -24:] == 3).all())
        q3, _ = bd.quantize_rows_int8(x)
        assert torch.equal(q3, bd.quantize_rows_int8(x0)[0])


def test_leading_axes_and_no_rows():
    x, r, gain = _make(23, 12, 160, "fp16")
    h, q, s = bd.add_rms_norm_int8(x.view(3, 4, 160), r.view(3, 4, 160), gain, 1e-6)
    h2, q2, s2 = bd.add_rms_norm_int8(x, r, gain, 1e-6)
    assert h.shape == q.shape == (3, 4, 160) and s.shape == (3, 4) and torch.equal(h.view(12, 160), h2) and torch.equal(q.view(12, 160), q2) and torch.equal(s.view(-1), s2)
    e = x[:0]
    assert bd.add_rms_norm(e, e, gain, 1e-6)[1].shape == (0, 160)
    assert bd.add_rms_norm_int8(e, None, gain, 1e-6)[2].shape == (0,) and bd.quantize_rows_int8(e)[0].shape == (0, 160)


def test_rows_agree_with_the_operators_that_they_join():
    """add_inplace_vec and rms_norm_rows: the same sum bit for bit, the norm to one step of the type where its FP32 value lies at a border."""
    x, r, gain = _make(29, 257, 1152, "bf16")
    h, y = bd.add_rms_norm(x, r, gain, 1e-6)
    two = x.clone()
    bd.add_inplace_vec(two, r)
    assert torch.equal(two, h)
    sep = bd.rms_norm_rows(two, gain, 1e-6)
    assert torch.all((sep.double() - y.double()).abs() <= torch.finfo(torch.bfloat16).eps * sep.double().abs())


def test_rows_past_two_to_the_31_elements():
    """The last rows of tensors of more than 2^31 elements: each row a view of a buffer with a large row stride."""
    cols, rows, stride = 1032, 70, 8 * 4_000_000
    buf = torch.zeros((rows - 1) * stride + cols, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, cols), (stride, 1))
    g = torch.Generator().manual_seed(2)
    x.copy_(torch.randn(rows, cols, generator=g).bfloat16())
    gain = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    q, s = bd.quantize_rows_int8(x)
    q2, s2 = bd.quantize_rows_int8(x.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    dense = x.contiguous()
    h, y = bd.add_rms_norm(x, dense, gain, 1e-6, sum_out=x)
    h2, y2 = bd.add_rms_norm(dense, dense, gain, 1e-6)
    assert torch.equal(h.contiguous(), h2) and torch.equal(y, y2)


def test_many_rows():
    """More rows than a launch has work groups of one row each."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((1 << 22) + 37, 8, generator=g, device="cuda").bfloat16()
    q, s = bd.quantize_rows_int8(x)
    assert torch.equal(q, _steps(x.float())[0]) and bool((s > 0).all())


def test_refusals():
    x, r, gain = _make(31, 4, 64, "bf16")
    for call, text in [
        (lambda: bd.add_rms_norm(x, r.half(), gain, 1e-6), "residual has dtype"),
        (lambda: bd.add_rms_norm(x, r[:3], gain, 1e-6), "residual has shape"),
        (lambda: bd.add_rms_norm(x, r, gain[:32], 1e-6), "gain"),
        (lambda: bd.add_rms_norm(x, None, gain, 1e-6, sum_out=x), "sum_out without a residual"),
        (lambda: bd.add_rms_norm(x, r, gain, -1.0), "eps"),
        (lambda: bd.add_rms_norm(x, r, gain, float("nan")), "eps"),
        (lambda: bd.add_rms_norm(x.cpu(), r, gain, 1e-6), "not on the GPU"),
        (lambda: bd.add_rms_norm(x.float(), None, gain.float(), 1e-6), "not supported"),
        (lambda: bd.add_rms_norm(x.t(), None, torch.ones(4, dtype=x.dtype, device="cuda"), 1e-6), "contiguous"),
        (lambda: bd.add_rms_norm(x[:, :60], None, gain[:60], 1e-6), "multiple of 8"),
        (lambda: bd.add_rms_norm(x[:, 4:36], None, gain[:32], 1e-6), "aligned"),
        (lambda: bd.add_rms_norm_int8(x, r, gain, 1e-6, scales=torch.empty(3, device="cuda")), "scales"),
        (lambda: bd.add_rms_norm_int8(x, r, gain, 1e-6, out=torch.empty_like(x)), "out has dtype"),
        (lambda: bd.add_rms_norm(x, r, gain, 1e-6, sum_out=(s := torch.empty_like(x)), out=s), "overlaps"),
        (lambda: bd.add_rms_norm_int8(x, r, gain, 1e-6, out=x.view(torch.int8)[:, :64]), "overlaps"),
        (lambda: bd.quantize_rows_int8(x, out=x.view(torch.int8)[:, 64:]), "overlaps"),
        (lambda: bd.quantize_rows_int8(x.float()), "not supported"),
        (lambda: bd.quantize_rows_int8(torch.empty(1, 65544, dtype=torch.half, device="cuda")), "65536"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_captured_rows_replay_like_eager_calls():
    x, r, gain = _make(37, 64, 6144, "bf16")
    h, q, s = torch.empty_like(x), torch.empty(64, 6144, dtype=torch.int8, device="cuda"), torch.empty(64, device="cuda")
    q2, s2 = torch.empty_like(q), torch.empty_like(s)

    def go():
        bd.add_rms_norm_int8(x, r, gain, 1e-6, sum_out=h, out=q, scales=s)
        bd.quantize_rows_int8(h, out=q2, scales=s2)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for i in range(4):
        x.copy_(torch.randn(64, 6144, generator=torch.Generator().manual_seed(i)).bfloat16())
        eager = [t.clone() for t in (*bd.add_rms_norm_int8(x, r, gain, 1e-6), *bd.quantize_rows_int8(bd.add_rms_norm(x, r, gain, 1e-6)[0]))]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((h, q, s, q2, s2), eager):
            assert torch.equal(got, want), i
