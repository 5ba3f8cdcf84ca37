"""linear_act against act(x w^T + b) + r in 64 bits: 16-bit operands, INT8 weights, INT8 rows and weights.

Bounds, for u = eps / 2 of the output type and S = sum |x w| (scaled as the sum is): the output is rounded once, u |y|; an FP32 sum of K
exact products in any order is at most K 2^-24 S off, INT32 sums are exact, the scales, the bias and the residual add at most 6 roundings of 2^-24 of
what they join; the activations have slopes up to 1.13 and are computed to 2e-5 of their value (exp2 of an argument of up to 2^5 that is
itself rounded: 2^5 2^-24 ln 2, and three more roundings; GELU's fit 1.5e-5)."""
import math

import pytest
import torch

import brodiffusion_amd as bd
from helpers import TORCH_DT

pytestmark = pytest.mark.gpu

KINDS = ["w16", "w8", "w8a8"]
# rows: one token, both sides of 16, 32 and 64, of a tile; features and contractions of one piece, of a stage, one piece more
SIZES = [(1, 8, 16), (1, 1160, 320), (1, 40, 4608), (2, 264, 1152), (15, 72, 208), (16, 1288, 64), (17, 48, 1168), (20, 640, 5120), (31, 96, 512), (33, 200, 144),
         (48, 1032, 640), (64, 136, 2240), (65, 520, 128), (77, 1280, 768), (130, 72, 48), (257, 264, 192), (300, 1160, 1168), (1031, 648, 1152), (2049, 392, 320)]


def make(seed, kind, M, N, K, dtype, bias=True, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TORCH_DT[dtype]

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    c = {"dt": dt, "K": K, "x_scales": None, "w_scales": None}
    if kind == "w8a8":
        c["x"] = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
        c["x_scales"] = (0.5 + torch.rand(M, generator=g, device="cuda")) / 74
    else:
        c["x"] = randn(M, K).to(dt)
    if kind == "w16":
        c["w"] = (randn(N, K) / math.sqrt(K)).to(dt)
    else:
        c["w"] = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        c["w_scales"] = (0.5 + torch.rand(N, generator=g, device="cuda")) / (74 * math.sqrt(K))
    c["bias"] = randn(N).to(dt) if bias else None
    c["residual"] = randn(M, N).to(dt) if residual else None
    return c


def call(c, act="none", **kw):
    a = dict(activation=act, residual=c["residual"], x_scales=c["x_scales"], w_scales=c["w_scales"], dtype=c["dt"])
    a.update(kw)
    return bd.linear_act(c["x"], c["w"], c["bias"], **a)


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def check(c, act, y, what=""):
    x, w = c["x"].double(), c["w"].double()
    if c["x_scales"] is not None:
        x = x * c["x_scales"].double()[:, None]
    if c["w_scales"] is not None:
        w = w * c["w_scales"].double()[:, None]
    v = x @ w.t()
    size = x.abs() @ w.abs().t()
    # (2^-53: what these sums here are off by; an INT8 sum of exactly zero is one that rounding leaves at 1e-17)
    err = ((0 if c["x_scales"] is not None else c["K"]) * 2.0 ** -24 + c["K"] * 2.0 ** -53) * size
    joined = v.abs()
    if c["bias"] is not None:
        v = v + c["bias"].double()
        joined = joined + c["bias"].double().abs()
    ref = _act(v, act)
    err = 1.13 * (err + 4 * 2.0 ** -24 * joined) + (2e-5 if act != "none" else 0.0) * ref.abs()
    if c["residual"] is not None:
        ref = ref + c["residual"].double()
        err = err + 2 * 2.0 ** -24 * (ref.abs() + c["residual"].double().abs())
    fi = torch.finfo(c["dt"])
    bound = ref.abs() * fi.eps / 2 + err * (1 + fi.eps) + fi.tiny * fi.eps
    off = (y.double() - ref).abs()
    assert y.dtype == c["dt"] and y.shape == ref.shape
    assert bool((off <= bound).all()), f"{what}: {float((off / bound).max())} of the bound at {int((off / bound).argmax())}"


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_act_sizes(dtype, kind, M, N, K):
    act = ["none", "gelu", "gelu_tanh", "silu"][(M + N // 8 + K // 8) % 4]
    c = make(M + N + K, kind, M, N, K, dtype)
    check(c, act, call(c, act), f"{kind} {M}x{N}x{K} {act}")


@pytest.mark.parametrize("kind", ["w16", "w8"])
@pytest.mark.parametrize("M,N,K", [(1, 24, 8), (3, 16, 24), (19, 72, 1160), (70, 136, 72), (513, 1288, 1288), (1031, 200, 648), (2100, 1160, 328)])
def test_contractions_of_odd_pieces(kind, M, N, K):
    """in_features that are multiples of 8 and not of 16."""
    c = make(M + N + K, kind, M, N, K, "fp16")
    check(c, "silu", call(c, "silu"), f"{kind} {M}x{N}x{K}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("M,N,K", [(5, 328, 640), (1100, 328, 640)])
def test_epilogues(kind, act, bias, residual, M, N, K):
    c = make(41, kind, M, N, K, "bf16", bias, residual)
    check(c, act, call(c, act), f"{kind} {act}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", [(4608, 1536, 1152), (4100, 4616, 640), (1, 16384, 6144), (24, 6144, 16384), (1, 1152, 131056), (600, 264, 16400)])
def test_large(kind, M, N, K):
    c = make(43, kind, M, N, K, "bf16")
    check(c, "gelu_tanh", call(c, "gelu_tanh"), f"{kind} {M}x{N}x{K}")


def test_int8_sums_are_exact_at_the_limit():
    """131056 products of -128 and -128 (the largest INT32 sum that there is) and of 127 and -128, against integers."""
    K = 131056
    for M in (1, 70):
        x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((16, K), -128, dtype=torch.int8, device="cuda")
        x[0], w[3] = 127, 127
        ones = torch.ones(M, device="cuda"), torch.full((16,), 2.0 ** -20, device="cuda")
        y = bd.linear_act(x, w, x_scales=ones[0], w_scales=ones[1], dtype=torch.bfloat16)
        want = (x.double() @ w.double().t() * 2.0 ** -20)
        assert torch.equal(y, want.float().bfloat16())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [3, 40, 500])
def test_strides_and_results_into_the_residual(kind, M):
    """x, w, the residual and the result as column slices of wider tensors; the result into the residual itself."""
    N, K = 200, 400
    c = make(47, kind, M, N, K, "fp16")
    want = call(c, "gelu")
    check(c, "gelu", want)

    def wide(t, pad):
        w = torch.full((t.shape[0], t.shape[1] + 2 * pad), 5, dtype=t.dtype, device="cuda")
        w[:, pad:-pad] = t
        return w, w[:, pad:-pad]

    d = dict(c)
    (_, d["x"]), (_, d["w"]), (rw, d["residual"]) = wide(c["x"], 16), wide(c["w"], 32), wide(c["residual"], 8)
    ow, o = wide(torch.zeros_like(c["residual"]), 24)
    assert call(d, "gelu", out=o) is o and torch.equal(o, want)
    assert bool((ow[:, :24] == 5).all()) and bool((ow[:, -24:] == 5).all())
    assert call(d, "gelu", out=d["residual"]) is d["residual"] and torch.equal(d["residual"], want)
    assert bool((rw[:, :8] == 5).all()) and bool((rw[:, -8:] == 5).all())


def test_without_an_epilogue_it_is_the_linear_layer():
    """linear_batched's values to half a step each: both round the same FP32 sum, added in another order."""
    for kind in ("w16", "w8"):
        c = make(53, kind, 300, 320, 640, "fp16", True, False)
        y = bd.linear_batched(c["w"], c["bias"], c["x"], W_scales=c["w_scales"])
        assert torch.all((y.double() - call(c).double()).abs() <= torch.finfo(torch.float16).eps * y.double().abs().clamp(min=2.0 ** -6))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [2, 90])
def test_values_that_are_not_finite(kind, M):
    """A NaN or infinity stays in its row (of x, of the scales, of the residual), and a row of scale NaN is NaN; no activation hides one."""
    for act in ("none", "gelu", "gelu_tanh", "silu"):
        c = make(59, kind, M, 40, 160, "bf16")
        if kind == "w8a8":
            c["x_scales"][1] = float("nan")
        else:
            c["x"][1, 7] = float("nan")
        c["residual"][0, 3] = float("inf")
        y = call(c, act)
        assert torch.isnan(y[1]).all() and y[0, 3] == float("inf")
        y[1], y[0, 3] = 0, 0
        assert torch.isfinite(y).all()


def test_large_arguments_of_the_activations():
    """Identity weights put the values through the activation: far left 0, far right the value."""
    v = torch.tensor([0.0, 1e-30, -1e-30, 1.0, -1.0, 5.0, -5.0, 12.0, -12.0, 30.0, -30.0, 1e4, -1e4, 1e15, -1e15, 3e38, -3e38], device="cuda")
    K = 32
    x = torch.zeros(len(v), K, device="cuda")
    x[:, 0] = v
    x, w = x.bfloat16(), torch.eye(K, device="cuda").bfloat16()
    for act in ("gelu", "gelu_tanh", "silu"):
        y = bd.linear_act(x, w, activation=act)[:, 0].double()
        r = x[:, 0].double()
        ref = _act(r, act).nan_to_num(0.0) if act != "gelu_tanh" else r * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (r + 0.044715 * r ** 3))
        assert torch.all((y - ref).abs() <= ref.abs() * 2.0 ** -8 * 1.01 + 1e-30), act


def test_leading_axes_and_no_rows():
    c = make(61, "w16", 12, 40, 64, "fp16")
    y = call(c, "silu")
    z = bd.linear_act(c["x"].view(3, 4, 64), c["w"], c["bias"], activation="silu", residual=c["residual"].view(3, 4, 40))
    assert z.shape == (3, 4, 40) and torch.equal(z.view(12, 40), y)
    assert bd.linear_act(c["x"][:0], c["w"], c["bias"]).shape == (0, 40)


def test_results_do_not_depend_on_the_rows_around_or_the_run():
    c = make(67, "w8a8", 40, 328, 640, "bf16")
    a = call(c, "gelu")
    assert all(torch.equal(a, call(c, "gelu")) for _ in range(3))


def test_a_block_half_of_8_bit_rows():
    """norm -> first product -> rows -> second product with the residual, as a decoder's MLP uses them, on one token, a draft and a prompt; eager,
    and captured and replayed, against the same steps in 64 bits from the integers on."""
    D, F = 640, 2560
    g = torch.Generator(device="cuda").manual_seed(71)
    gain = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
    w1, w2 = (torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((F, D), (D, F)))
    s1, s2 = torch.full((F,), 1 / (74 * D ** 0.5), device="cuda"), torch.full((D,), 1 / (74 * F ** 0.5), device="cuda")
    b1, b2 = torch.randn(F, generator=g, device="cuda").bfloat16(), torch.randn(D, generator=g, device="cuda").bfloat16()
    for M in (1, 20, 333):
        x, r = (torch.randn(M, D, generator=g, device="cuda").bfloat16() for _ in range(2))

        def half():
            h, q, s = bd.add_rms_norm_int8(x, r, gain, 1e-6)
            u = bd.linear_act(q, w1, b1, activation="gelu", x_scales=s, w_scales=s1)
            q2, sq = bd.quantize_rows_int8(u)
            return h, q, s, u, q2, sq, bd.linear_act(q2, w2, b2, residual=h, x_scales=sq, w_scales=s2)

        half()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = half()
        for i in range(3):
            x.copy_(torch.randn(M, D, generator=g, device="cuda"))
            h, q, s, u, q2, sq, y = half()
            c = {"dt": torch.bfloat16, "K": D, "x": q, "x_scales": s, "w": w1, "w_scales": s1, "bias": b1, "residual": None}
            check(c, "gelu", u, "first product")
            c = {"dt": torch.bfloat16, "K": F, "x": q2, "x_scales": sq, "w": w2, "w_scales": s2, "bias": b2, "residual": h}
            check(c, "none", y, "second product")
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for got, want in zip(captured, (h, q, s, u, q2, sq, y)):
                assert torch.equal(got, want), (M, i)


def test_on_another_stream():
    c = make(73, "w8a8", 33, 328, 640, "fp16")
    want = call(c, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(c, "silu")
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    c = make(79, "w16", 4, 40, 64, "fp16")
    x, w, b, r = c["x"], c["w"], c["bias"], c["residual"]
    i8 = make(83, "w8a8", 4, 40, 64, "fp16")
    both = torch.zeros(5, 40, dtype=x.dtype, device="cuda")
    for f, text in [
        (lambda: bd.linear_act(x, w, b, activation="relu"), "activation"),
        (lambda: bd.linear_act(x, w[:, :56], b), "W is"),
        (lambda: bd.linear_act(x, w.bfloat16(), b), "W has dtype"),
        (lambda: bd.linear_act(x, w, b.bfloat16()), "bias"),
        (lambda: bd.linear_act(x, w, b, residual=r[:3]), "residual has shape"),
        (lambda: bd.linear_act(x, w, b, residual=r.bfloat16()), "residual has dtype"),
        (lambda: bd.linear_act(x, w, b, dtype=torch.bfloat16), "is not X's"),
        (lambda: bd.linear_act(x, w, b, x_scales=i8["x_scales"]), "INT8 weights"),
        (lambda: bd.linear_act(x, i8["w"], b, w_scales=i8["w_scales"][:8]), "w_scales"),
        (lambda: bd.linear_act(i8["x"], i8["w"], x_scales=i8["x_scales"], w_scales=i8["w_scales"]), "need a dtype"),
        (lambda: bd.linear_act(i8["x"], i8["w"], x_scales=i8["x_scales"][:2], w_scales=i8["w_scales"], dtype=torch.half), "x_scales"),
        (lambda: bd.linear_act(i8["x"], i8["w"], x_scales=i8["x_scales"], w_scales=i8["w_scales"], dtype=torch.float32), "not supported"),
        (lambda: bd.linear_act(i8["x"][:, :56], i8["w"][:, :56], x_scales=i8["x_scales"], w_scales=i8["w_scales"], dtype=torch.half), "multiple of 16"),
        (lambda: bd.linear_act(x[:, :60], w[:, :60]), "multiple of 8"),
        (lambda: bd.linear_act(x, w[:36]), "of 8"),
        (lambda: bd.linear_act(x.cpu(), w), "not on the GPU"),
        (lambda: bd.linear_act(x, w, out=r.t()), "shape"),
        (lambda: bd.linear_act(x, w, residual=both[:4], out=both[1:]), "overlaps"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            f()
