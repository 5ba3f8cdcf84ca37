"""gate_add_norm with vectors as models cut them, slices of a modulation's columns, through both forms of the call: bit for bit what contiguous copies of them give."""
import pytest
import torch

import brodiffusion_amd as bd
import brodiffusion_amd.ops as ops

pytestmark = pytest.mark.gpu


class _Declines:
    def __getattr__(self, name):
        return lambda *a: None


class _Only:
    """The native form alone: a call that it leaves to the Python form fails"""

    def __init__(self, native):
        self.native = native

    def gate_add_norm(self, *a):
        r = self.native.gate_add_norm(*a)
        assert r is not None
        return r


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("items,tokens,cols", [(2, 37, 1160), (3, 1, 64), (1, 5, 520)])
def test_slices_of_a_modulation(monkeypatch, native, items, tokens, cols):
    g = torch.Generator().manual_seed(items + tokens)
    x, b = (torch.randn(items, tokens, cols, generator=g).bfloat16().cuda() for _ in range(2))
    mods = [torch.randn(*s, 6 * cols, generator=g).bfloat16().cuda() for s in ((items, tokens), (items, 1), (items,), ())]
    bd.gate_add_norm(x, b)      # (binds the native module)
    monkeypatch.setattr(ops, "_native", _Only(ops._native) if native else _Declines())
    for mod in mods:
        parts = [mod[..., i * cols:(i + 1) * cols] for i in (2, 0, 5)]
        got = bd.gate_add_norm(x, b, norm="layer", **dict(zip(("gate", "scale", "shift"), parts)))
        each = [p.reshape(*p.shape[:-1], *(1,) * (3 - p.dim()), cols) if p.dim() in (1, 3) else p[:, None] for p in parts]
        each = [p.expand(items, tokens, cols).contiguous() for p in each]
        want = bd.gate_add_norm(x, b, norm="layer", **dict(zip(("gate", "scale", "shift"), each)))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    flat = mods[0].view(-1, 6 * cols)
    got = bd.gate_add_norm(x.view(-1, cols), b.view(-1, cols), gate=flat[:, :cols], norm="layer", shift=flat[:, None, cols:2 * cols])
    want = bd.gate_add_norm(x.view(-1, cols), b.view(-1, cols), gate=flat[:, :cols].contiguous(), norm="layer", shift=flat[:, cols:2 * cols].contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_vectors_without_rows_or_apart_by_less_than_one():
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda")
    mod = torch.zeros(2, 4, 384, dtype=x.dtype, device="cuda")
    for v in (mod[:0, 0, :64], mod[:, :0, :64], mod[:, :3, :64], mod[:, :1, :64].expand(2, 3, 64), mod[0, 0, :66].as_strided((2, 64), (2, 1))):
        with pytest.raises(RuntimeError, match="gate_add_norm: gate (must be contiguous along columns|is)"):
            bd.gate_add_norm(x, x, gate=v)
    with pytest.raises(RuntimeError, match="gate_add_norm: gate is"):
        bd.gate_add_norm(x.view(6, 64), x.view(6, 64), gate=mod[:0, 0, :64])
