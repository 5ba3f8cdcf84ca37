"""gate_add_norm's Python form without a GPU: which vectors it takes and what it hands to the C entry (a stand-in that notes its arguments)."""
import pytest
import torch

from brodiffusion_amd import ops


@pytest.fixture
def call(monkeypatch):
    got = []

    class Library:
        @staticmethod
        def mi_gate_add_norm_forward(args):
            got.append(args._obj)
            return 0
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops.capi, "lib", lambda: Library)
    monkeypatch.setattr(ops, "_native", type("Declines", (), {"gate_add_norm": staticmethod(lambda *a: None)}))

    def run(x, **kw):
        got.clear()
        ops.gate_add_norm(x, torch.zeros_like(x), **kw)
        return got[0]
    return run


def _t(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("name", ["gate", "scale", "shift"])
def test_no_vectors_for_some_rows(call, name):
    """A slice without rows has no memory, and a null pointer would say that there is no gate"""
    mod = _t(2, 64)
    for x, v in ((_t(6, 64), mod[:0]), (_t(6, 64), mod[:0, None]), (_t(2, 3, 64), mod[:0]), (_t(2, 3, 64), _t(2, 0, 64))):
        with pytest.raises(RuntimeError, match=f"gate_add_norm: {name} is"):
            call(x, norm="layer", **{name: v})
    for x in (_t(0, 64), _t(0, 3, 64)):      # (no rows: nothing to be done)
        assert call(x, norm="layer", **{name: mod[:0]}).rows == 0
    assert call(_t(2, 0, 64), norm="layer", **{name: mod}).rows == 0
