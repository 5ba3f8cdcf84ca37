"""gate_add_norm against its formulas in 64 bits: widths of one chunk, one past a wavefront's, one past a work group's and the largest; each norm on either side;
vectors of all rows, of each item and of each row; rows that are zero, constant, far from zero or not finite; strides; outputs that are their inputs.

Tolerances, with e = 2^-24 (half an FP32 step). The kernels add at most 64 terms in a row, then in a tree, so a sum of them is off by at most 80 e of the sum of
magnitudes. RMS: the mean square by 82 e of itself, its inverse root by half of that and 2 units: REL. Layer: the mean by D = 81 e mean|v|, every difference
by D and a rounding; the mean square of the differences, which add up to nothing, by D^2 and 84 e of itself. Behind that each product or sum is one
rounding e of its result. h is then rounded to T (half a step), and y is held to the formula on the h that came back."""
import pytest
import torch

import brodiffusion_amd as bd
from helpers import TORCH_DT

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
SIZES = [(1, 8), (3, 64), (5, 512), (4, 520), (7, 1160), (333, 2240), (2, 2568), (9, 3080), (2, 4096), (3, 4104), (1, 6144), (5, 10248), (2, 16384), (3, 16392),
         (2, 33000), (1, 65536), (1031, 1152), (1100, 16392)]


def _normed(v, kind, eps, gain):
    """(value, bound of its error) of the norm of v (FP64)"""
    if kind == "none":
        n, err = v, torch.zeros_like(v)
    else:
        d = 0.0
        if kind == "layer":
            d = 81 * E * v.abs().mean(dim=-1, keepdim=True)
            v = v - v.mean(dim=-1, keepdim=True)
        ms = v.square().mean(dim=-1, keepdim=True)
        inv = (ms + eps).rsqrt()
        inv_err = 0.5 * (84 * E * ms + d ** 2) / (ms + eps) + 4 * E
        n = v * inv
        err = n.abs() * (inv_err * 1.01 + 3 * E) + d * inv * 1.01
    if gain is None:
        return n, err
    n = n * gain
    return n, err * gain.abs() + n.abs() * E


def _check(x, branch, dtype, h, y, *, gate=None, post="none", post_gain=None, post_eps=1e-6, alpha=1.0, norm="rms", gain=None, scale=None, shift=None, eps=1e-6):
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny
    wide = lambda t: None if t is None else t.double()
    if branch is not None:
        b, err = _normed(branch.double(), post, post_eps, wide(post_gain))
        if gate is not None:
            b, err = b * gate.double(), err * gate.double().abs() + (b * gate.double()).abs() * E
        alpha = float(torch.tensor(alpha, dtype=torch.float32))
        ref = alpha * x.double() + b
        err = err + (ref.abs() + err) * E
        assert torch.all((h.double() - ref).abs() <= err * (1 + half) + ref.abs() * half + tiny * half)
    else:
        assert h is x
    if norm == "none":
        assert y is None
        return
    n, err = _normed(h.double(), norm, eps, wide(gain))
    if scale is not None:
        s = 1 + scale.double()
        n, err = n * s, err * s.abs() + 2 * E * (n * s).abs()
    if shift is not None:
        n = n + shift.double()
        err = err + (n.abs() + err) * E
    assert torch.all((y.double() - n).abs() <= err * (1 + half) + n.abs() * half + tiny * half)


def _make(seed, dtype, *shape):
    g = torch.Generator().manual_seed(seed)
    loud = torch.exp(torch.randn(shape[-1], generator=g))
    x, b = ((torch.randn(*shape, generator=g) * loud + 0.5).to(TORCH_DT[dtype]).cuda() for _ in range(2))

    def vec(*s, base=0.0):
        return (base + 0.3 * torch.randn(*s, generator=g)).to(TORCH_DT[dtype]).cuda()
    return x, b, vec


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("post,norm", [("none", "layer"), ("rms", "rms"), ("layer", "rms"), ("rms", "none"), ("none", "rms"), ("layer", "layer")])
def test_sizes(dtype, rows, cols, post, norm):
    x, b, vec = _make(7 * rows + cols, dtype, rows, cols)
    kw = dict(gate=vec(cols), alpha=0.8125)
    if post == "rms":
        kw["post_gain"] = vec(cols, base=1.0)
    if norm == "rms":
        kw["gain"] = vec(cols, base=1.0)
    if norm == "layer":
        kw["scale"], kw["shift"] = vec(cols), vec(cols)
    alpha = kw.pop("alpha")
    h, y = bd.gate_add_norm(x, b, post=post, norm=norm, residual_scale=alpha, **kw)
    _check(x, b, x.dtype, h, y, post=post, norm=norm, alpha=alpha, **kw)


@pytest.mark.parametrize("rows,cols", [(1, 64), (37, 1152), (300, 2240)])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_no_branch(rows, cols, norm):
    x, _, vec = _make(rows, "bf16", rows, cols)
    kw = dict(scale=vec(cols), shift=vec(cols), norm=norm)
    h, y = bd.gate_add_norm(x, None, eps=1e-5, **kw)
    _check(x, None, x.dtype, h, y, eps=1e-5, **kw)


def test_two_eps_and_plain_sum():
    x, b, _ = _make(5, "fp16", 9, 1152)
    h, y = bd.gate_add_norm(x, b, post="rms", post_eps=0.5, eps=0.0)
    _check(x, b, x.dtype, h, y, post="rms", post_eps=0.5, eps=0.0)
    h, y = bd.gate_add_norm(x, b, norm="none")
    assert y is None and torch.equal(h, (x.float() + b.float()).half())
    h, y = bd.gate_add_norm(x, b, norm="none", residual_scale=0.0)
    assert torch.equal(h, b)
    h, y = bd.gate_add_norm(x, b)
    s, z = bd.add_rms_norm(x, b, torch.ones(1152, dtype=x.dtype, device="cuda"), 1e-6)
    assert torch.equal(h, s) and torch.equal(y, z)      # the same sums in the same order


@pytest.mark.parametrize("items,tokens,cols", [(1, 5, 64), (3, 1, 1152), (9, 37, 2240), (2, 700, 520)])
def test_vectors_of_items_and_rows(items, tokens, cols):
    x, b, vec = _make(items, "bf16", items, tokens, cols)
    chunks = vec(items, 6 * cols)                                    # a modulation's row cut in six
    gate, scale, shift = (chunks[:, i * cols:(i + 1) * cols] for i in (5, 0, 2))
    wide = lambda t: t[:, None, :]
    h, y = bd.gate_add_norm(x, b, gate=gate, scale=scale, shift=shift, norm="layer")
    _check(x, b, x.dtype, h, y, gate=wide(gate), scale=wide(scale), shift=wide(shift), norm="layer")
    for g, s, t in ((wide(gate), wide(scale), wide(shift)), (gate.contiguous(), scale, wide(shift).contiguous())):
        h2, y2 = bd.gate_add_norm(x, b, gate=g, scale=s, shift=t, norm="layer")
        assert torch.equal(h, h2) and torch.equal(y, y2)
    # rows of all items behind one another
    h2, y2 = bd.gate_add_norm(x.view(-1, cols), b.view(-1, cols), gate=gate, scale=scale, shift=shift, norm="layer")
    assert torch.equal(h.view(-1, cols), h2) and torch.equal(y.view(-1, cols), y2)
    # one shared, one of each item, one of each row
    shared, each = vec(cols), vec(items, tokens, cols)
    h, y = bd.gate_add_norm(x, b, gate=shared, scale=each, shift=shift, norm="rms")
    _check(x, b, x.dtype, h, y, gate=shared, scale=each, shift=wide(shift), norm="rms")
    h, y = bd.gate_add_norm(x, b, gate=each, scale=shared, norm="rms")
    _check(x, b, x.dtype, h, y, gate=each, scale=shared, norm="rms")
    # results do not depend on the other rows
    one, two = bd.gate_add_norm(x[:1, :1].contiguous(), b[:1, :1].contiguous(), gate=each[:1, :1].contiguous(), scale=shared, norm="rms")
    if tokens * items < 1024:
        assert torch.equal(one, h[:1, :1]) and torch.equal(two, y[:1, :1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_strides_and_outputs_that_are_inputs(dtype):
    rows, cols = 37, 1160
    x, b, vec = _make(3, dtype, rows, cols)
    gate, gain = vec(cols), vec(cols, base=1.0)
    h, y = bd.gate_add_norm(x, b, gate=gate, post="rms", gain=gain)
    big = torch.full((4, rows, cols + 24), 7.0, dtype=x.dtype, device="cuda")
    big[0, :, 8:cols + 8], big[1, :, :cols] = x, b
    out = bd.gate_add_norm(big[0, :, 8:cols + 8], big[1, :, :cols], gate=gate, post="rms", gain=gain, sum_out=big[2, :, 16:cols + 16], out=big[3, :, 24:])
    assert torch.equal(out[0], h) and torch.equal(out[1], y)
    assert torch.all(big[2, :, :16] == 7) and torch.all(big[2, :, cols + 16:] == 7) and torch.all(big[3, :, :24] == 7)
    assert torch.all(big[0, :, :8] == 7) and torch.all(big[0, :, cols + 8:] == 7) and torch.all(big[1, :, cols:] == 7)
    for first, second in (("x", "b"), ("b", "x")):
        t = {"x": x.clone(), "b": b.clone()}
        out = bd.gate_add_norm(t["x"], t["b"], gate=gate, post="rms", gain=gain, sum_out=t[first], out=t[second])
        assert out[0] is t[first] and torch.equal(t[first], h) and torch.equal(t[second], y)


def test_odd_rows():
    """Rows of zeros, constant rows, rows far from zero, tiny and not finite ones, each among others"""
    cols = 1152
    x, b, vec = _make(11, "bf16", 8, cols)
    x[0], b[0] = 0, 0
    x[1], b[1] = 3.0, 0
    x[2] = (1000 + torch.randn(cols)).to(x.dtype)
    x[3], b[3] = 2.0 ** -64, 2.0 ** -64
    gate = vec(cols)
    for norm in ("rms", "layer"):
        h, y = bd.gate_add_norm(x, b, gate=gate, post="layer", norm=norm, eps=1e-6)
        _check(x, b, x.dtype, h, y, gate=gate, post="layer", norm=norm)
        assert torch.all(y[0] == 0) and torch.isfinite(y).all()
    h, y = bd.gate_add_norm(x[3:4], b[3:4] * 0, eps=0.0)      # without eps: mean squares below FP32's smallest normal number
    assert torch.all(y == 1)
    x[5, 17], b[6, 9], x[7, 0] = float("inf"), float("nan"), float("-inf")
    for norm in ("rms", "layer"):
        h2, y2 = bd.gate_add_norm(x, b, gate=gate, post="layer", norm=norm)
        keep = [0, 1, 2, 3, 4]
        hk, yk = bd.gate_add_norm(x[keep], b[keep], gate=gate, post="layer", norm=norm)
        assert torch.equal(h2[keep], hk) and torch.equal(y2[keep], yk)
        assert torch.isnan(y2[6]).all() and torch.isnan(h2[6]).all()
        assert torch.isinf(h2[5, 17]) and torch.isnan(y2[5, 17]) and not torch.isfinite(y2[7, 0])


def test_no_rows_and_untouched_rows():
    cols = 64
    e = torch.empty(0, cols, dtype=torch.bfloat16, device="cuda")
    h, y = bd.gate_add_norm(e, e, gate=torch.ones(cols, dtype=e.dtype, device="cuda"))
    assert h.shape == (0, cols) and y.shape == (0, cols)
    x, b, _ = _make(2, "bf16", 5, cols)
    h, y = (torch.full((8, cols), 9.0, dtype=x.dtype, device="cuda") for _ in range(2))
    bd.gate_add_norm(x, b, sum_out=h[:5], out=y[:5])
    assert torch.all(h[5:] == 9) and torch.all(y[5:] == 9)


def test_far_rows():
    """Rows and vectors 2^30 elements apart: offsets past 32 bits"""
    cols, apart = 1152, (1 << 30) + 8
    x, b, vec = _make(6, "bf16", 4, cols)
    gate, shift = vec(4, cols), vec(2, cols)
    want = bd.gate_add_norm(x, b, gate=gate, post="rms", norm="layer", shift=shift)
    ins, outs = (torch.empty(3 * apart + 4 * cols, dtype=x.dtype, device="cuda") for _ in range(2))
    at = lambda i, rows=4: (ins if i < 4 else outs).as_strided((rows, cols), (apart, 1), i % 4 * cols)
    for i, t in enumerate((x, b, gate, shift)):
        at(i, t.shape[0]).copy_(t)
    h, y = bd.gate_add_norm(at(0), at(1), gate=at(2), post="rms", norm="layer", shift=at(3, 2), sum_out=at(4), out=at(5))
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_other_stream_and_graph():
    x, b, vec = _make(4, "fp16", 333, 1152)
    gate = vec(1152)
    want = bd.gate_add_norm(x, b, gate=gate, post="rms")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = bd.gate_add_norm(x, b, gate=gate, post="rms")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x2, b2 = x.clone(), b.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = bd.gate_add_norm(x2, b2, gate=gate, post="rms")
    for i in range(3):
        x2.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = bd.gate_add_norm(x2, b2, gate=gate, post="rms")
        assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_native_and_python_forms_agree(monkeypatch):
    import brodiffusion_amd.ops as ops
    x, b, vec = _make(6, "bf16", 2, 19, 520)
    calls = [dict(), dict(gate=vec(520), norm="none"), dict(gate=vec(2, 520), post="rms", post_gain=vec(520), gain=vec(520)),
             dict(scale=vec(2, 1, 520), shift=vec(520), norm="layer", residual_scale=0.5, eps=1e-3, post="layer", post_eps=1e-2)]
    native = [bd.gate_add_norm(x, b, **kw) for kw in calls] + [bd.gate_add_norm(x, None, norm="layer")]

    class Declines:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_native", Declines())
    python = [bd.gate_add_norm(x, b, **kw) for kw in calls] + [bd.gate_add_norm(x, None, norm="layer")]
    for n, p in zip(native, python):
        assert all((u is None and v is None) or torch.equal(u, v) for u, v in zip(n, p))


@pytest.mark.parametrize("kw,said", [
    (dict(post="l2"), "none of"), (dict(norm="batch"), "none of"), (dict(gate="half"), "gate must hold"), (dict(gate="rows3"), "gate is"), (dict(gate="float"), "gate must hold"),
    (dict(gain="half"), "gain must hold"), (dict(post_gain="cols"), "post_gain without"), (dict(norm="none", gain="cols"), "without a norm"), (dict(norm="none", shift="cols"), "without a norm"),
    (dict(branch=None, gate="cols"), "without a branch"), (dict(branch=None, norm="none"), "neither"), (dict(branch="half"), "shape"), (dict(sum_out="half"), "shape"),
    (dict(out="float"), "dtype"), (dict(out="part"), "overlaps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(post_eps=float("inf")), "eps"),
    (dict(residual_scale=float("nan")), "residual_scale"), (dict(gate="expanded"), "contiguous"), (dict(sum_out="gate", gate="same"), "overlaps gate"), (dict(branch="cpu"), "not on the GPU")])
def test_refusals(kw, said):
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(2 * 2 * 4 * 64, dtype=x.dtype, device="cuda")
    things = {"half": torch.zeros(2, 4, 32, dtype=x.dtype, device="cuda"), "rows3": torch.zeros(3, 64, dtype=x.dtype, device="cuda"), "float": torch.zeros(2, 4, 64, device="cuda"),
              "cols": torch.zeros(64, dtype=x.dtype, device="cuda"), "part": None, "expanded": torch.zeros(1, 64, dtype=x.dtype, device="cuda").expand(2, 64),
              "cpu": torch.zeros(2, 4, 64, dtype=x.dtype), "gate": flat[:512].view(2, 4, 64), "same": flat[64:128]}
    args = {k: things[v] if isinstance(v, str) and v in things else v for k, v in kw.items()}
    if kw.get("out") == "part":
        x, args["out"] = flat[:512].view(2, 4, 64), flat[64:576].view(2, 4, 64)
    branch = args.pop("branch", torch.zeros_like(x))
    with pytest.raises(RuntimeError, match="gate_add_norm") as e:
        bd.gate_add_norm(x, branch, **args)
    assert said in str(e.value), str(e.value)
