"""The new operator calls in native code (host/py_ops.cpp) against the Python code behind them (ops.py): the same results, the same objects handed
back, and only what is plainly valid taken."""
import pytest
import torch

import brodiffusion_amd as bd
from brodiffusion_amd import ops
from test_linear_act_gpu import call, make

pytestmark = pytest.mark.gpu


class _Declines:
    def __getattr__(self, name):
        return lambda *a: None


def _both(monkeypatch, f):
    native = f()
    with monkeypatch.context() as m:
        m.setattr(ops, "_native", _Declines())
        python = f()
    return native, python


def _same(a, b):
    a, b = (a, b) if isinstance(a, tuple) else ((a,), (b,))
    assert len(a) == len(b)
    for u, v in zip(a, b):
        assert u.shape == v.shape and u.dtype == v.dtype and u.stride() == v.stride() and torch.equal(u, v)


@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 64), (64,), (0, 64)])
def test_rows_both_ways(monkeypatch, shape):
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(*shape, generator=g).bfloat16().cuda() for _ in range(2))
    gain = torch.rand(64, generator=g).bfloat16().cuda()
    for f in (lambda: bd.add_rms_norm(x, r, gain, 1e-6), lambda: bd.add_rms_norm(x, None, gain, 1e-6), lambda: bd.add_rms_norm_int8(x, r, gain, 1e-6),
              lambda: bd.add_rms_norm_int8(x, None, gain, 1e-6), lambda: bd.quantize_rows_int8(x)):
        _same(*_both(monkeypatch, f))
    if len(shape) == 2 and shape[0]:
        wide = torch.zeros(5, 96, dtype=torch.bfloat16, device="cuda")
        wide[:, 16:80] = x
        _same(*_both(monkeypatch, lambda: bd.add_rms_norm_int8(wide[:, 16:80], r, gain, 1e-6)))
    out, q, s = torch.empty_like(x), torch.empty(shape, dtype=torch.int8, device="cuda"), torch.empty(shape[:-1], device="cuda")
    for way in range(2):
        with monkeypatch.context() as m:
            if way:
                m.setattr(ops, "_native", _Declines())
            h, y = bd.add_rms_norm(x, r, gain, 1e-6, sum_out=out)
            assert h is out
            h, y = bd.add_rms_norm(x, None, gain, 1e-6, out=out)
            assert h is x and y is out
            h, a, b = bd.add_rms_norm_int8(x, None, gain, 1e-6, out=q, scales=s)
            assert h is x and a is q and b is s
            a, b = bd.quantize_rows_int8(x, out=q, scales=s)
            assert a is q and b is s


@pytest.mark.parametrize("kind", ["w16", "w8", "w8a8"])
def test_linear_both_ways(monkeypatch, kind):
    c = make(3, kind, 6, 40, 64, "fp16")
    for act in ("none", "gelu", "gelu_tanh", "silu"):
        _same(*_both(monkeypatch, lambda: call(c, act)))
    _same(*_both(monkeypatch, lambda: bd.linear_act(c["x"], c["w"], c["bias"], x_scales=c["x_scales"], w_scales=c["w_scales"])))
    _same(*_both(monkeypatch, lambda: bd.linear_act(c["x"].view(2, 3, 64), c["w"], None, residual=c["residual"].view(2, 3, 40), x_scales=c["x_scales"], w_scales=c["w_scales"])))
    _same(*_both(monkeypatch, lambda: bd.linear_act(c["x"][0], c["w"], c["bias"], x_scales=None if kind != "w8a8" else c["x_scales"][:1], w_scales=c["w_scales"])))
    out = torch.empty(6, 40, dtype=torch.half, device="cuda")
    for way in range(2):
        with monkeypatch.context() as m:
            if way:
                m.setattr(ops, "_native", _Declines())
            assert call(c, out=out) is out


def test_refusals_are_worded_by_either():
    """Calls that the native half declines raise the Python half's error; those that the library refuses carry its own words."""
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="linear_act: mi_linear_act_forward: in_features"):
        bd.linear_act(x[:, :60].contiguous(), torch.zeros(8, 60, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="add_rms_norm: mi_add_rms_norm_forward: cols"):
        bd.add_rms_norm(x[:, :60].contiguous(), None, torch.zeros(60, dtype=torch.bfloat16, device="cuda"), 1e-6)
    with pytest.raises(RuntimeError, match="linear_act: activation"):
        bd.linear_act(x, torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda"), activation=None)
    with pytest.raises(RuntimeError, match="must have columns"):
        bd.quantize_rows_int8(torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError):
        bd.linear_act(torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 0, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError):
        bd.linear_act(x, torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda"))
