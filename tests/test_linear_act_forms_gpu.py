"""linear_act on every kernel that its rules choose from: each tile form of the rings with whole and partial last stages (the form asked of the rule
itself), and each work-group shape for few rows. Operands with poisoned borders (NaN, or 127 in INT8) and results in wider buffers;
tests/test_linear_act_gpu.py derives the bounds."""
import ctypes as C
import os

import pytest
import torch

import brodiffusion_amd as bd
from brodiffusion_amd import build
from test_linear_act_gpu import call, check, make
from test_linear_pipe_gpu import FORMS

pytestmark = pytest.mark.gpu


def _form(M, N, K, int8):
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    return C.CDLL(build.FORMS_LIB).linear_form((C.c_int * 3)(M, N, K), 1, int8, 0, bd.device_info()["compute_units"])


def _off_form(M, N, K, row, int8=0):
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    splits = C.c_int()
    return C.CDLL(build.FORMS_LIB).linear_parts(M, N, K, row, int8, bd.device_info()["compute_units"], C.byref(splits)), splits.value


def _poisoned(t, pad):
    wide = torch.full((t.shape[0], t.shape[1] + pad), 127 if t.dtype == torch.int8 else float("nan"), dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _run(kind, M, N, K, dtype, act, what, on_lines=False):
    c = make(M + N + K, kind, M, N, K, dtype)
    # (INT8 weights of a contraction that is a multiple of 8 only: rows on 8-byte addresses)
    pads = 16 if kind == "w8a8" else 8, 16 if kind != "w8" or K % 16 == 0 else 8
    if on_lines:       # rows of both operands begin on 128-byte lines
        line = 128 if kind == "w8a8" else 64
        pads = (line - K % line, line - K % line)
    c["x"], c["w"] = _poisoned(c["x"], pads[0]), _poisoned(c["w"], pads[1])
    wide = torch.full((M + 1, N + 8), 7.0, dtype=c["dt"], device="cuda")
    out = wide[:M, :N]
    call(c, act, out=out)
    check(c, act, out, what)
    assert bool((wide[M:] == 7).all()) and bool((wide[:, N:] == 7).all())


# (every one has more rows than the kernel for few rows takes)
RINGS = [f for f in FORMS if f[1] == 0 and f[3] == 1] + [(0, 0, 11, 1, 2188, 5392, 512), (0, 0, 11, 1, 2188, 5392, 576)]


@pytest.mark.parametrize("int8,geglu,form,n,M,N,K", RINGS)
def test_every_ring_form(int8, geglu, form, n, M, N, K):
    dtype, act = ("fp16", "bf16")[K // 64 % 2], ("none", "gelu", "gelu_tanh", "silu")[M % 4]
    for more in (0, 8, 40, 48):       # (a partial stage changes no form: the rule counts whole ones)
        assert _form(M, N, K + more, int8) == form
        _run("w8" if int8 else "w16", M, N, K + more, dtype, act, f"{form} +{more}", on_lines=True)
        if not int8:
            _run("w8a8", M, N, 2 * (K + more), dtype, act, f"{form} INT8 +{more}", on_lines=True)


# 16-bit and INT8 operands whose rows begin off lines: every form of that rule, with one to many stages (and as many partial ones), by rows of every
# distance to a line, aligned to 16 bytes as they must be
OFF_FORMS = [(0, 70, 328, 200), (0, 37, 1160, 328), (1, 33, 4616, 200), (2, 200, 13000, 200), (3, 1500, 8200, 584), (3, 1500, 16392, 1000), (4, 768, 648, 4616), (5, 33, 8200, 200), (5, 130, 4616, 1288),
             (6, 77, 8200, 200), (7, 77, 13000, 200), (8, 200, 8200, 200), (8, 200, 8200, 1288), (9, 200, 13000, 328), (9, 200, 13000, 1288), (10, 500, 8200, 200), (10, 500, 8200, 1288)]


@pytest.mark.parametrize("form,M,N,K", OFF_FORMS)
def test_every_form_of_rows_off_lines(form, M, N, K):
    for i, beyond in enumerate((8, 24, 32, 56)):      # elements of a row stride beyond whole lines
        k = K + (0, 8, 16, 48)[i]
        pad = (beyond - k) % 64 or 64
        assert _off_form(M, N, k, k + pad) == (form, 1)
        dtype, act = ("fp16", "bf16")[i % 2], ("none", "gelu", "gelu_tanh", "silu")[i]
        for kind, two in (("w16", 1), ("w8a8", 2)):
            c = make(M + N + k, kind, M, N, two * k, dtype, residual=i != 2)
            c["x"], c["w"] = _poisoned(c["x"], two * pad), _poisoned(c["w"], two * pad)
            wide = torch.full((M + 1, N + 8), 7.0, dtype=c["dt"], device="cuda")
            call(c, act, out=wide[:M, :N])
            check(c, act, wide[:M, :N], f"{kind} {form} {k}")
            assert bool((wide[M:] == 7).all()) and bool((wide[:, N:] == 7).all())


OFF8_FORMS = [(0, 33, 328, 200), (1, 33, 8200, 200), (2, 77, 8200, 200), (3, 200, 8200, 200), (4, 77, 13000, 328), (5, 130, 8200, 4616), (6, 768, 8200, 200), (6, 768, 8200, 584),
              (7, 200, 13000, 200), (7, 200, 13000, 328)]


@pytest.mark.parametrize("form,M,N,K", OFF8_FORMS)
def test_every_form_of_int8_weights_off_lines(form, M, N, K):
    """(K is an odd multiple of 8: every second row of the weights begins within a piece of 16 bytes)"""
    for i, pad in enumerate((0, 16, 32, 64)):
        for k in (K, K + 8):
            assert _off_form(M, N, k, k + pad, 1) == (form, 1)
            c = make(M + N + k + pad, "w8", M, N, k, ("fp16", "bf16")[i % 2], residual=i != 2)
            if pad:
                c["x"], c["w"] = _poisoned(c["x"], pad), _poisoned(c["w"], pad)
            wide = torch.full((M + 1, N + 8), 7.0, dtype=c["dt"], device="cuda")
            act = ("none", "gelu", "gelu_tanh", "silu")[i]
            call(c, act, out=wide[:M, :N])
            check(c, act, wide[:M, :N], f"{form} {k} + {pad}")
            assert bool((wide[M:] == 7).all()) and bool((wide[:, N:] == 7).all())


@pytest.mark.parametrize("kind,two", [("w16", 1), ("w8a8", 2)])
def test_rows_off_lines_give_the_bits_of_rows_on_them(kind, two):
    """The order of the sums does not hang on where rows begin; also with one operand's rows on lines, or both tensors' first bytes off them."""
    M, N, K = 300, 1160, 712
    c = make(9, kind, M, N, two * K, "bf16")
    ref = None
    for xp, wp, shift in ((56, 56, 0), (8, 8, 0), (56, 16, 0), (16, 56, 0), (56, 56, 8), (24, 40, 24), (0, 0, 0)):
        def placed(t, pad):
            wide = torch.full((t.shape[0] * (t.shape[1] + two * pad) + two * shift,), 127 if t.dtype == torch.int8 else float("nan"), dtype=t.dtype, device="cuda")
            v = wide[two * shift:].view(t.shape[0], t.shape[1] + two * pad)[:, :t.shape[1]]
            v.copy_(t)
            return v
        got = call({**c, "x": placed(c["x"], xp), "w": placed(c["w"], wp)}, "silu")
        if ref is None:
            ref = got
            check(c, "silu", got, "on lines")
        assert torch.equal(got, ref), (xp, wp, shift)


# rows at the ends of each class; features: narrow (also fewer than one work group's), up to 16 per compute unit, three and four blocks, wide
@pytest.mark.parametrize("kind", ["w16", "w8", "w8a8"])
@pytest.mark.parametrize("N", [24, 2040, 2056, 4096, 6136, 8200, 16392])
@pytest.mark.parametrize("K", [80, 1168, 4880, 5184])
def test_every_shape_of_few_rows(kind, N, K):
    for M in (1, 4, 5, 8, 9, 16, 17, 24, 25, 32):
        _run(kind, M, N, K + (8 if kind == "w8" and M % 2 else 0), ("fp16", "bf16")[M % 2], ("none", "gelu", "gelu_tanh", "silu")[M % 4], f"{M} rows")


def test_few_rows_give_the_same_bits_alone_and_together():
    """Rows of one class: a row's result does not depend on the other rows or on how many there are."""
    for kind in ("w16", "w8", "w8a8"):
        c = make(91, kind, 16, 6136, 1168, "bf16")
        whole = call(c, "silu")
        for first, last in ((9, 16), (0, 9)):
            d = {**c, "x": torch.cat([c["x"][first:last], c["x"][:9]])[:16].contiguous(), "residual": torch.cat([c["residual"][first:last], c["residual"][:9]])[:16].contiguous()}
            if c["x_scales"] is not None:
                d["x_scales"] = torch.cat([c["x_scales"][first:last], c["x_scales"][:9]])[:16].contiguous()
            assert torch.equal(call(d, "silu")[:last - first], whole[first:last])


@pytest.mark.parametrize("M", [3, 40])
def test_weights_past_two_to_the_31_elements(M):
    N, K = 65544, 32784
    g = torch.Generator(device="cuda").manual_seed(7)
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    s = torch.full((N,), 1 / (74 * K ** 0.5), device="cuda")
    x = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.full((M,), 1 / 74, device="cuda")
    y = bd.linear_act(x, w, x_scales=xs, w_scales=s, dtype=torch.bfloat16)
    xb = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    yb = bd.linear_act(xb, w, w_scales=s)
    for cols in (slice(0, 40), slice(N - 40, N)):
        c = {"dt": torch.bfloat16, "K": K, "x": x, "x_scales": xs, "w": w[cols], "w_scales": s[cols], "bias": None, "residual": None}
        check(c, "none", y[:, cols].contiguous(), "INT8 rows")
        check({**c, "x": xb, "x_scales": None}, "none", yb[:, cols].contiguous(), "16-bit rows")


def test_results_past_two_to_the_31_elements():
    M, N, K = 70001, 32768, 64
    c = make(97, "w16", M, 8, K, "bf16", False, False)
    w = torch.randn(N, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    y.fill_(1)
    bd.linear_act(c["x"], w, activation="gelu", residual=y, out=y)
    for rows in (slice(0, 70), slice(M - 70, M)):
        d = {"dt": torch.bfloat16, "K": K, "x": c["x"][rows], "x_scales": None, "w": w, "w_scales": None, "bias": None, "residual": torch.ones(70, N, dtype=torch.bfloat16, device="cuda")}
        check(d, "gelu", y[rows], "rows")


@pytest.mark.parametrize("kind", ["w16", "w8", "w8a8"])
@pytest.mark.parametrize("M,N,K", [(40, 72, 144), (40, 200, 1168)])
def test_rows_too_far_apart_for_the_rings(kind, M, N, K):
    """A row stride of x past 32-bit offsets within a tile: the form with tiles through registers."""
    c = make(101, kind, M, N, K, "fp16")
    stride = 4_194_304 * (2 if kind == "w8a8" else 1)
    buf = torch.zeros((M - 1) * stride + K, dtype=c["x"].dtype, device="cuda")
    x = buf.as_strided((M, K), (stride, 1))
    x.copy_(c["x"])
    c["x"] = x
    check(c, "gelu", call(c, "gelu"), kind)
