"""linear_int4 against its formula in 64 bits, on every path: rows, features and contractions that end inside a tile, an operand, a block and a group; groups of
32 to more than a block; with and without zero points; strides; outputs that are the residual.

Tolerance: a group's sum has exact products (4 + 11 bits) and starts at -z sum(x), itself a sum in FP32. At any order each of its additions rounds by at most
2^-23 (the matrix instructions may cut off) of a partial sum no larger than A = sum (q + 2 z) |x|, and there are up to 2 (g + 4) of them for g <= 128
elements of a group in a block. Groups, parts of a contraction (8) and bias meet by additions that round to 2^-24 of at most B = sum |q - z| s |x| + |bias|, three
roundings each. The activations (slopes up to 1.13) are within 2e-5 of their value. The result is rounded to the type once: half a step. Beside that bound, which adds up
magnitudes, the whole result is held to half a step in its norm: what a rounding of exact values gives is 0.58 of that at most."""
import ctypes as C
import math

import pytest
import torch

import brodiffusion_amd as bd
from brodiffusion_amd import _capi as capi
from brodiffusion_amd import build
from helpers import TORCH_DT

pytestmark = pytest.mark.gpu


def _checkpoint(g, n, k, group, zeros, t):
    groups = -(-k // group)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).cuda()
    scales = ((0.5 + torch.rand(n, groups, generator=g)) / (4.6 * math.sqrt(k))).to(t).cuda()
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8).cuda() if zeros else None
    return q, scales, z


def _act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.erfc(v * -(0.5 ** 0.5)) / 2
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def _reference(x, q, scales, z, group, bias, act, residual):
    """(value, bound of the error ahead of the last rounding)"""
    n, k = q.shape[0], 2 * q.shape[1]
    w = torch.stack((q & 15, q >> 4), dim=2).view(n, k).double()
    wide = lambda t: t.double().repeat_interleave(group, dim=1)[:, :k]
    zero, s, x = (wide(z) if z is not None else torch.full_like(w, 8.0)), wide(scales), x.double()
    v = x @ ((w - zero) * s).t()
    a = x.abs() @ ((w + 2 * zero) * s).t()
    b = x.abs() @ ((w - zero).abs() * s).t()
    if bias is not None:
        v, b = v + bias.double(), b + bias.double().abs()
    err = 2 * (min(group, 128) + 4) * 2.0 ** -23 * a + 3 * (scales.shape[1] + -(-k // 128) + 10) * 2.0 ** -24 * b
    v = _act(v, act)
    if act != "none":
        err = 1.13 * err + 2e-5 * v.abs()
    if residual is not None:
        v = v + residual.double()
        err = err + 2.0 ** -24 * (v.abs() + err)
    return v, err


def _check(y, ref, err):
    half, tiny = torch.finfo(y.dtype).eps / 2, torch.finfo(y.dtype).tiny
    off = (y.double() - ref).abs()
    assert torch.all(off <= err * (1 + half) + ref.abs() * half + tiny * half), float((off - ref.abs() * half).max())
    if ref.numel() > 64:
        assert off.norm() <= half * ref.norm()


def _case(dtype, m, k, n, group, zeros, bias, act, residual, seed=0):
    g = torch.Generator().manual_seed(1000 * m + 10 * k + n + seed)
    t = TORCH_DT[dtype]
    x = (torch.randn(m, k, generator=g) + 0.2).to(t).cuda()
    q, scales, z = _checkpoint(g, n, k, group, zeros, t)
    b = torch.randn(n, generator=g).to(t).cuda() if bias else None
    r = torch.randn(m, n, generator=g).to(t).cuda() if residual else None
    y = bd.linear_int4(x, bd.pack_int4(q, scales, z, group=group), b, activation=act, residual=r)
    assert y.shape == (m, n) and y.dtype == t
    _check(y, *_reference(x, q, scales, z, group, b, act, r))


SIZES = [(1, 8, 8), (1, 128, 16), (3, 120, 24), (16, 136, 72), (17, 256, 264), (33, 1160, 136), (64, 2240, 1152), (5, 4104, 40), (1, 6144, 2048), (65, 8, 8), (65, 264, 72),
         (77, 4608, 1152), (130, 1160, 520), (333, 2240, 264), (128, 384, 64)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True), (256, True), (1152, False)])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(dtype, m, k, n, group, zeros):
    _case(dtype, m, k, n, group, zeros, bias=n % 16 == 8, act=("none", "gelu", "gelu_tanh", "silu")[(m + group // 32) % 4], residual=k % 16 == 8)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False), (128, True)])
@pytest.mark.parametrize("m,k,n", [(1, 1152, 16392), (16, 2056, 8200), (20, 1160, 16384), (40, 520, 16392), (1031, 520, 8200), (4608, 264, 2056), (300, 136, 33032)])
def test_wide_and_long(dtype, m, k, n, group, zeros):
    _case(dtype, m, k, n, group, zeros, bias=True, act="gelu_tanh", residual=True)


FEW16, FEW32, FEW64, TILE32x64, TILE32x128, TILE64x128, TILE64x192, TILE96x192, TILE64x256 = range(9)
# (rows, contraction, features) by group, work group, and whether the contraction is given in shares
PROBLEMS = {
    128: {(FEW16, 0): (40, 136, 72), (FEW16, 1): (64, 8200, 8), (FEW32, 0): (40, 136, 2056), (FEW32, 1): (17, 16392, 264), (FEW64, 0): (777, 520, 264),
         (FEW64, 1): (1, 16392, 4104), (TILE32x64, 0): (333, 8, 4104), (TILE32x64, 1): (500, 8200, 264), (TILE32x128, 0): (40, 1160, 8200), (TILE32x128, 1): (64, 3088, 4104),
         (TILE64x128, 0): (1500, 520, 2056), (TILE64x128, 1): (2049, 16392, 72), (TILE64x192, 0): (2049, 8, 8200), (TILE64x192, 1): (4096, 8200, 136), (TILE96x192, 0): (2049, 264, 4104),
         (TILE96x192, 1): (3000, 16392, 136), (TILE64x256, 0): (777, 136, 16392), (TILE64x256, 1): (64, 16392, 8200)},
    64: {(FEW16, 0): (17, 136, 136), (FEW16, 1): (17, 16392, 8), (FEW32, 0): (40, 136, 2056), (FEW32, 1): (17, 8200, 520), (FEW64, 0): (40, 520, 4104),
         (FEW64, 1): (1, 16392, 4104), (TILE32x64, 0): (40, 136, 4104), (TILE32x64, 1): (64, 4616, 2056), (TILE32x128, 0): (2049, 136, 1160), (TILE32x128, 1): (17, 3088, 16392),
         (TILE64x128, 0): (777, 1160, 4104), (TILE64x128, 1): (4096, 16392, 72), (TILE64x192, 0): (500, 136, 16392), (TILE64x192, 1): (4096, 8200, 136), (TILE96x192, 0): (1500, 520, 2056),
         (TILE96x192, 1): (1031, 8200, 1160)},
    32: {(FEW16, 0): (1, 264, 1160), (FEW16, 1): (40, 8200, 8), (FEW32, 0): (5, 520, 4104), (FEW32, 1): (17, 8200, 520), (TILE32x64, 0): (64, 136, 4104),
         (TILE32x64, 1): (500, 8200, 136), (TILE32x128, 0): (100, 520, 16392), (TILE32x128, 1): (333, 16392, 2056), (TILE64x128, 0): (1031, 264, 4104), (TILE64x128, 1): (100, 8200, 8200),
         (TILE64x192, 1): (40, 16392, 16392), (TILE96x192, 0): (4096, 520, 2056), (TILE96x192, 1): (1031, 3088, 4104)}}


def _launch(m, k, n, group, lent=(1 << 64) - 1):
    shares = C.c_int()
    return C.CDLL(build.FORMS_LIB).int4_form_test(m, n, k, C.c_long(k), group, bd.device_info()["compute_units"], C.c_ulong(lent), C.byref(shares)), shares.value


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,form,shared", [(g, *f) for g in PROBLEMS for f in PROBLEMS[g]])
def test_every_form(dtype, zeros, group, form, shared):
    """Every kernel instance, with the contraction whole and in shares, on problems that end inside its work groups, its steps and their groups"""
    m, k, n = PROBLEMS[group][form, shared]
    got, shares = _launch(m, k, n, group)
    assert got == form and (shares > 1) == bool(shared)
    _case(dtype, m, k, n, group, zeros, bias=True, act="silu", residual=True)


def _args(x, w, y, scratch=None):
    a = capi.MiLinearInt4Args()
    a.struct_size, a.dtype = C.sizeof(a), capi.MI_DTYPE_BF16
    a.x, a.w, a.scales, a.y = x.data_ptr(), w.packed.data_ptr(), w.scales.data_ptr(), y.data_ptr()
    a.rows, a.in_features, a.out_features, a.group = x.shape[0], w.in_features, w.out_features, w.group
    a.stream = torch.cuda.current_stream().cuda_stream
    if scratch is not None:
        a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel()
    return a


@pytest.mark.parametrize("m", [1, 40, 200])
def test_scratch(m):
    """As much as is asked for, less, none, and more; what lies behind it stays"""
    g = torch.Generator().manual_seed(m)
    k, n = 16392, 264
    q, scales, _ = _checkpoint(g, n, k, 128, False, torch.bfloat16)
    w = bd.pack_int4(q, scales)
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    ref = _reference(x, q, scales, None, 128, None, "none", None)
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    need = int(capi.lib().mi_linear_int4_scratch_bytes(C.byref(_args(x, w, y))))
    assert need == 4 * m * n * _launch(m, k, n, 128)[1] > 4 * m * n
    memory = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    for lent in (need, need - 4, need // 2, 4 * m * n, 0, need + 4096):
        memory.fill_(77)
        y.fill_(9)
        a = _args(x, w, y, memory)
        a.scratch_bytes = lent
        assert capi.lib().mi_linear_int4_forward(C.byref(a)) == 0
        _check(y, *ref)
        assert torch.all(memory[4 * m * n * _launch(m, k, n, 128, lent)[1] if lent >= 8 * m * n else 0:] == 77)
    assert torch.equal(bd.linear_int4(x, w), y)


@pytest.mark.parametrize("m", [1, 20, 40, 100, 1031])
def test_every_weight_and_its_place(m):
    """One nonzero x per row: the results are single weights, exactly"""
    k, n, group = 1160, 72, 32
    g = torch.Generator().manual_seed(m)
    q, _, z = _checkpoint(g, n, k, group, True, torch.bfloat16)
    scales = (2.0 ** torch.randint(-3, 4, (n, -(-k // group)), generator=g)).to(torch.bfloat16).cuda()
    w = torch.stack((q & 15, q >> 4), dim=2).view(n, k).float() - z.float().repeat_interleave(group, dim=1)[:, :k]
    w = w * scales.float().repeat_interleave(group, dim=1)[:, :k]
    packed = bd.pack_int4(q, scales, z, group=group)
    for first in range(0, k, m):
        rows = min(m, k - first)
        x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
        x[torch.arange(rows), first + torch.arange(rows)] = 1
        y = bd.linear_int4(x, packed)
        assert torch.equal(y[:rows].float(), w.t()[first:first + rows]) and torch.all(y[rows:] == 0)
        if m == 1 and first > 300:
            break


@pytest.mark.parametrize("m", [3, 60, 200])
def test_strides_and_leading_axes(m):
    g = torch.Generator().manual_seed(m)
    k, n = 1160, 136
    q, scales, z = _checkpoint(g, n, k, 64, True, torch.float16)
    wide_q = torch.full((n, k // 2 + 12), 255, dtype=torch.uint8, device="cuda")
    wide_q[:, 4:k // 2 + 4] = q
    w, w2 = bd.pack_int4(q, scales, z, group=64), bd.pack_int4(wide_q[:, 4:k // 2 + 4], scales, z, group=64)
    assert torch.equal(w.packed, w2.packed)
    x, r = torch.randn(m, k, generator=g).half().cuda(), torch.randn(m, n, generator=g).half().cuda()
    want = bd.linear_int4(x, w, residual=r)
    big = torch.full((3, m + 2, k + 16), 7.0, dtype=torch.float16, device="cuda")
    big[0, 1:m + 1, 8:k + 8], big[1, 1:m + 1, :n] = x, r
    got = bd.linear_int4(big[0, 1:m + 1, 8:k + 8], w, residual=big[1, 1:m + 1, :n], out=big[2, 1:m + 1, 16:n + 16])
    assert torch.equal(got, want)
    assert torch.all(big[2, 0] == 7) and torch.all(big[2, m + 1] == 7) and torch.all(big[2, :, :16] == 7) and torch.all(big[2, :, n + 16:] == 7)
    r2 = r.clone()
    assert bd.linear_int4(x, w, residual=r2, out=r2) is r2 and torch.equal(r2, want)
    y = bd.linear_int4(x.view(1, m, 1, k), w, residual=r.view(1, m, 1, n))
    assert y.shape == (1, m, 1, n) and torch.equal(y.view(m, n), want)
    assert bd.linear_int4(x[:0], w).shape == (0, n)


@pytest.mark.parametrize("m,k", [(4, 520), (50, 520), (90, 520), (300, 520), (4, 8200), (300, 8200)])
def test_rows_that_are_not_finite_stay_alone(m, k):
    g = torch.Generator().manual_seed(m)
    n = 264
    q, scales, z = _checkpoint(g, n, k, 128, False, torch.bfloat16)
    w = bd.pack_int4(q, scales, z)
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    want = bd.linear_int4(x, w)
    x[1, 519], x[3, 0], x[2, 130] = float("inf"), float("nan"), float("-inf")
    y = bd.linear_int4(x, w)
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[1:4]).all()


def test_far_rows():
    """Rows 2^24 elements apart: offsets past 32 bits, in x and in y"""
    g = torch.Generator().manual_seed(1)
    k, n, m, apart = 136, 72, 70, 1 << 24
    q, scales, z = _checkpoint(g, n, k, 64, True, torch.bfloat16)
    w = bd.pack_int4(q, scales, z, group=64)
    store = torch.empty((m - 1) * apart + 8192, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((m, k), (apart, 1))
    x.copy_(torch.randn(m, k, generator=g))
    _check(bd.linear_int4(x, w), *_reference(x.contiguous(), q, scales, z, 64, None, "none", None))
    y = store.as_strided((m, n), (apart, 1), 4096)
    bd.linear_int4(x.contiguous(), w, out=y)
    _check(y.contiguous(), *_reference(x.contiguous(), q, scales, z, 64, None, "none", None))


def test_rows_as_far_apart_as_tiles_reach():
    """The largest row stride whose tiles have 32-bit offsets (csrc/linear_int4_forms.h): 96 rows of it are 512 bytes short of 2^31"""
    g = torch.Generator().manual_seed(8)
    k, n, m, apart = 136, 4104, 101, 11184808
    q, scales, _ = _checkpoint(g, n, k, 128, False, torch.float16)
    w = bd.pack_int4(q, scales)
    store = torch.empty((m - 1) * apart + k, dtype=torch.float16, device="cuda")
    x = store.as_strided((m, k), (apart, 1))
    x.copy_(torch.randn(m, k, generator=g))
    _check(bd.linear_int4(x, w), *_reference(x.contiguous(), q, scales, None, 128, None, "none", None))


def test_calls_on_two_streams_at_once():
    """Calls whose contraction is in shares, in turn on two streams without waiting for each other: each has memory of its own"""
    g = torch.Generator().manual_seed(9)
    q, scales, z = _checkpoint(g, 264, 16392, 64, True, torch.bfloat16)
    w = bd.pack_int4(q, scales, z, group=64)
    xs = [torch.randn(m, 16392, generator=g).bfloat16().cuda() for m in (1, 40, 200, 17)]
    want = [bd.linear_int4(x, w) for x in xs]
    assert all(_launch(x.shape[0], 16392, 264, 64)[1] > 1 for x in xs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append(bd.linear_int4(xs[i % 4 if i < 20 else (i * 7 // 2) % 4], w))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4 if i < 20 else (i * 7 // 2) % 4])


def test_other_stream_and_graphs():
    g = torch.Generator().manual_seed(2)
    for m, k in ((1, 1160), (40, 1160), (200, 1160), (1, 8200), (200, 8200)):
        q, scales, z = _checkpoint(g, 520, k, 64, True, torch.float16)
        w = bd.pack_int4(q, scales, z, group=64)
        x = torch.randn(m, k, generator=g).half().cuda()
        want = bd.linear_int4(x, w, activation="gelu")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = bd.linear_int4(x, w, activation="gelu")
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        x2 = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = bd.linear_int4(x2, w, activation="gelu")
        for i in range(3):
            x2.copy_(x * (1 + i))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, bd.linear_int4(x2, w, activation="gelu"))


def test_native_and_python_forms_agree(monkeypatch):
    import brodiffusion_amd.ops as ops
    g = torch.Generator().manual_seed(3)
    q, scales, z = _checkpoint(g, 72, 264, 32, True, torch.bfloat16)
    w, w2 = bd.pack_int4(q, scales, z, group=32), bd.pack_int4(q, scales, None, group=32)
    x, r, b = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((2, 5, 264), (2, 5, 72), (72,)))
    calls = [((x, w), {}), ((x, w2, b), dict(activation="silu")), ((x, w), dict(residual=r)), ((x.view(10, 264), w, b), dict(residual=r.view(10, 72), activation="gelu"))]
    native = [bd.linear_int4(*a, **kw) for a, kw in calls]

    class Declines:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_native", Declines())
    for n, (a, kw) in zip(native, calls):
        assert torch.equal(n, bd.linear_int4(*a, **kw))


def test_a_block_as_it_is_used():
    """Norm, 4-bit projections with activation, and the next block's norm with the gated residual, captured together"""
    g = torch.Generator().manual_seed(4)
    t, d, hidden, items, tokens = torch.bfloat16, 1152, 4608, 2, 37
    q1, s1, _ = _checkpoint(g, hidden, d, 128, False, t)
    q2, s2, z2 = _checkpoint(g, d, hidden, 64, True, t)
    w1, w2 = bd.pack_int4(q1, s1), bd.pack_int4(q2, s2, z2, group=64)
    x, att = (torch.randn(items, tokens, d, generator=g).to(t).cuda() for _ in range(2))
    mod = (0.3 * torch.randn(items, 6 * d, generator=g)).to(t).cuda()
    gate1, shift, scale, gate2 = (mod[:, i * d:(i + 1) * d] for i in (2, 3, 4, 5))

    def block(x, att):
        h, y = bd.gate_add_norm(x, att, gate=gate1, norm="layer", scale=scale, shift=shift)
        u = bd.linear_int4(y, w1, activation="gelu_tanh")
        v = bd.linear_int4(u, w2)
        return h, y, u, v, *bd.gate_add_norm(h, v, gate=gate2, norm="layer")

    h, y, u, v, h2, y2 = block(x, att)
    _check(u.view(-1, hidden), *_reference(y.view(-1, d), q1, s1, None, 128, None, "gelu_tanh", None))
    _check(v.view(-1, d), *_reference(u.view(-1, hidden), q2, s2, z2, 64, None, "none", None))
    assert torch.equal(h2, (h.float() + (v.float() * gate2.float()[:, None])).to(t)) or (h2.float() - h.float() - v.float() * gate2.float()[:, None]).abs().max() < 0.1
    x2, att2 = x.clone(), att.clone()
    block(x2, att2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = block(x2, att2)
    for i in range(3):
        x2.copy_(x * (0.5 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, block(x2, att2)))


@pytest.mark.parametrize("group", [64, 256])
def test_packed_weights_are_copies(group):
    q, scales, z = _checkpoint(torch.Generator().manual_seed(6), 48, 256, group, True, torch.float16)
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(7)).half().cuda()
    w = bd.pack_int4(q, scales, z, group=group)
    y = bd.linear_int4(x, w)
    for t in (q, scales, z):
        t.zero_()
    assert torch.equal(bd.linear_int4(x, w), y) and y.abs().max() > 0


def test_refusals():
    g = torch.Generator().manual_seed(5)
    q, scales, z = _checkpoint(g, 16, 264, 64, True, torch.bfloat16)
    w = bd.pack_int4(q, scales, z, group=64)
    x = torch.zeros(3, 264, dtype=torch.bfloat16, device="cuda")
    import dataclasses
    for args, kw, said in [
            ((q.to(torch.int8), scales), {}, "uint8"), ((q, scales), dict(group=48), "group"), ((q, scales), dict(group=0), "group"), ((q, scales), dict(group=128), "scales are"),
            ((q, scales.float()), dict(group=64), "dtype"), ((q, scales, z.int()), dict(group=64), "zeros"), ((q, scales, z[:, :2]), dict(group=64), "zeros"),
            ((q[:, :131], scales), dict(group=64), "multiples of 8"), ((q[:12], scales[:12]), dict(group=64), "multiples of 8"), ((q.t(), scales), {}, "contiguous"),
            ((q.cpu(), scales), {}, "not on the GPU")]:
        with pytest.raises(RuntimeError, match="pack_int4") as e:
            bd.pack_int4(*args, **kw)
        assert said in str(e.value), str(e.value)
    flat = torch.zeros(3 * 264 + 3 * 16, dtype=x.dtype, device="cuda")
    for args, kw, said in [
            ((x, q), {}, "pack_int4 returns"), ((x[:, :256], w), {}, "in_features"), ((x.half(), w), {}, "scales"), ((x.float(), w), {}, "dtype"), ((x, w), dict(activation="relu"), "none of"),
            ((x, w, torch.zeros(8, dtype=x.dtype, device="cuda")), {}, "bias"), ((x, w), dict(residual=x), "residual"), ((x, w), dict(out=x[:, :16].float()), "out"),
            ((x, dataclasses.replace(w, group=48)), {}, "scales"), ((x, dataclasses.replace(w, group=66, scales=w.scales[:4].contiguous(), zeros=None)), {}, "group"),
            ((x, dataclasses.replace(w, packed=w.packed[:-1])), {}, "packed"), ((x, dataclasses.replace(w, zeros=w.zeros[:2])), {}, "zeros"),
            ((x, dataclasses.replace(w, scales=w.scales.cpu())), {}, "not on the GPU"), ((flat[:792].view(3, 264), w), dict(out=flat[784:832].view(3, 16)), "overlaps x")]:
        with pytest.raises(RuntimeError, match="linear_int4") as e:
            bd.linear_int4(*args, **kw)
        assert said in str(e.value), str(e.value)
