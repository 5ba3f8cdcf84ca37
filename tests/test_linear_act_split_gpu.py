"""linear_act where several work groups share a tile's contraction (mi_linear_act_scratch_bytes > 0): every tile form of the rule and numbers of
parts from 2 to 16, with and without the scratch; captured and replayed; bounds as in tests/test_linear_act_gpu.py."""
import ctypes as C
import os

import pytest
import torch

import brodiffusion_amd as bd
from brodiffusion_amd import _capi as capi
from brodiffusion_amd import build
from test_linear_act_gpu import call, check, make

pytestmark = pytest.mark.gpu


def _parts(M, N, K, int8):
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    splits = C.c_int()
    form = C.CDLL(build.FORMS_LIB).linear_parts(M, N, K, K, int8, bd.device_info()["compute_units"], C.byref(splits))
    return form, splits.value


def _args(c, act, out):
    M, K, N = *c["x"].shape, c["w"].shape[0]
    a = capi.MiLinearActArgs()
    a.struct_size = C.sizeof(a)
    a.dtype = capi.MI_DTYPE_BF16 if c["dt"] == torch.bfloat16 else capi.MI_DTYPE_F16
    a.rows, a.in_features, a.out_features = M, K, N
    a.x, a.w, a.y = c["x"].data_ptr(), c["w"].data_ptr(), out.data_ptr()
    for name in ("bias", "residual", "x_scales", "w_scales"):
        if c[name] is not None:
            setattr(a, name, c[name].data_ptr())
    a.activation = ["none", "gelu", "gelu_tanh", "silu"].index(act)
    a.stream = torch.cuda.current_stream().cuda_stream
    return a


# rows, features, contraction of 16-bit operands, and the form and parts that the rule gives them on 256 compute units
PLAIN = [(33, 72, 4608, 0, 16), (33, 520, 4608, 0, 6), (130, 520, 6400, 2, 8), (33, 704, 6400, 2, 16), (33, 2248, 8960, 2, 6), (100, 2248, 8960, 2, 3), (33, 6144, 16384, 2, 2),
         (65, 1640, 16384, 4, 8), (200, 2248, 12800, 7, 6), (65, 6144, 16384, 7, 4), (333, 1000, 16384, 7, 8), (200, 648, 16384, 4, 8), (65, 2240, 15936, 4, 6)]
W8 = [(33, 72, 3200, 0, 12), (33, 1000, 3200, 0, 4), (33, 360, 8960, 1, 16), (33, 6144, 6400, 1, 2), (65, 2248, 6400, 1, 3), (65, 1640, 12800, 3, 8), (65, 2248, 8960, 3, 6),
      (65, 3600, 8960, 4, 6), (130, 6144, 16384, 4, 2)]


@pytest.mark.parametrize("kind,M,N,K,form,splits", [("w16", *p) for p in PLAIN] + [("w8a8", *p) for p in PLAIN] + [("w8", *p) for p in W8])
def test_parts(kind, M, N, K, form, splits):
    assert _parts(M, N, K, kind == "w8") == (form, splits)
    # (whole stages, a partial last one and rows off lines, INT8 weights on 8-byte rows; twice the contraction of INT8 operands is the same stages)
    for more in (0, 8, 40):
        k = 2 * (K + more) if kind == "w8a8" else K + more
        splits = _parts(M, N, K + more, kind == "w8")[1]       # (rows off 128-byte lines: a table of their own)
        assert splits > 1
        c = make(M + N + K + more, kind, M, N, k, "bf16" if more else "fp16", residual=more != 8)
        act = ("none", "gelu", "silu")[more % 3]
        wide = torch.full((M + 1, N), 7.0, dtype=c["dt"], device="cuda")
        a = _args(c, act, wide[:M])
        need = capi.lib().mi_linear_act_scratch_bytes(C.byref(a))
        assert need >= M * N * splits * 4
        # guarded on both sides: nothing beyond what was asked for is written
        scratch = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        a.scratch, a.scratch_bytes = scratch.data_ptr() + 256, need
        assert capi.lib().mi_linear_act_forward(C.byref(a)) == 0, capi.last_error()
        check(c, act, wide[:M], f"{splits} parts")
        assert bool((wide[M:] == 7).all()) and bool((scratch[:256] == 77).all()) and bool((scratch[256 + need:] == 77).all())
        # a scratch that is too small is not used, and the whole tiles' result is another rounding of the same sums
        whole = torch.empty_like(wide)
        b = _args(c, act, whole[:M])
        scratch[:] = 77
        b.scratch, b.scratch_bytes = scratch.data_ptr() + 256, need - 16
        assert capi.lib().mi_linear_act_forward(C.byref(b)) == 0, capi.last_error()
        check(c, act, whole[:M], "whole")
        assert bool((scratch == 77).all())
        if kind == "w8a8":
            assert torch.equal(whole[:M], wide[:M])
        # the Python layer lends the scratch itself; into the residual, where there is one
        same = call(c, act, **({"out": c["residual"]} if c["residual"] is not None else {}))
        assert torch.equal(same, wide[:M])


def test_captured_parts_replay_like_eager_calls():
    """Two graphs captured one after the other and replayed on two streams at once: each has parts of its own."""
    cs = [make(s, "w16", 46, 368, 16000, "bf16") for s in (1, 2)]
    for c in cs:
        assert _parts(46, 368, 16000, 0)[1] > 1
        call(c, "gelu")
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cs], []
    for g, c in zip(graphs, cs):
        with torch.cuda.graph(g):
            outs.append(call(c, "gelu"))
    streams = [torch.cuda.Stream() for _ in cs]
    for i in range(4):
        for j, c in enumerate(cs):
            c["x"].copy_(torch.randn(46, 16000, generator=torch.Generator().manual_seed(10 * i + j)))
        want = [call(c, "gelu") for c in cs]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), i


def test_two_streams_at_once():
    cs = [make(s, "w8", 46, 368, 16000, "fp16") for s in (3, 4)]
    want = [call(c, "silu") for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for c, s, g in zip(cs, streams, got):
            with torch.cuda.stream(s):
                g.append(call(c, "silu"))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(o, w) for o in g)


def test_no_scratch_for_calls_that_use_none():
    c = make(5, "w16", 4, 368, 16000, "bf16")
    lib = capi.lib()
    assert lib.mi_linear_act_scratch_bytes(C.byref(_args(c, "none", c["residual"]))) == 0      # few rows
    c = make(6, "w16", 300, 512, 512, "bf16")
    a = _args(c, "none", c["residual"])
    assert lib.mi_linear_act_scratch_bytes(C.byref(a)) == 0      # a short contraction
    a.in_features = 12
    assert lib.mi_linear_act_scratch_bytes(C.byref(a)) == 0      # refused
    assert lib.mi_linear_act_scratch_bytes(None) == 0
    a = _args(c, "none", c["residual"])
    a.scratch, a.scratch_bytes = c["x"].data_ptr() + 8, 1 << 20
    assert lib.mi_linear_act_forward(C.byref(a)) == -1 and "scratch" in capi.last_error()
