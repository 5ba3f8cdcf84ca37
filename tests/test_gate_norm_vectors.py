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


def test_vectors_cut_out_of_a_modulation(call):
    """One vector a token, or an image, as a slice of a wider tensor: any row stride that all of them share"""
    cols, x = 64, _t(2, 3, 64)
    tokens, images, rows = _t(2, 3, 6 * cols), _t(2, 1, 6 * cols), _t(6, 6 * cols)
    part = lambda t: t[..., 2 * cols:3 * cols]
    for rows_of, v, each, stride in (
            (x, part(tokens), 1, 384), (x, part(tokens)[:, :1], 3, 1152), (x, part(images), 3, 384), (x.view(6, 64), part(rows), 1, 384), (x.view(6, 64), part(tokens)[:, 0], 3, 1152),
            (x.view(2, 3, 1, 64), part(tokens)[:, :, None], 1, 384), (x.view(2, 3, 1, 64), part(tokens), 1, 384), (x.view(1, 6, 64), part(rows)[None], 1, 384), (x, part(images).view(2, 64), 3, 384),
            (x, part(tokens)[:1, :1], 0, 64), (x[:1], part(tokens)[1:, :, :], 1, 384), (x[:1], part(tokens).transpose(0, 1)[:1, :1], 0, 64)):
        a = call(rows_of, gate=v)
        assert a.gate == v.data_ptr() and a.gate_rows == each and (each == 0 or a.gate_row_stride == stride)
    for rows_of, v in (
            (x[:1], part(tokens)), (x, part(_t(2, 4, 6 * cols))[:, :3]), (x, part(tokens)[:, :1].expand(2, 3, 64)), (x, _t(2, 64, 3).transpose(1, 2)),
            (x, _t(3, 2, 64).transpose(0, 1)), (_t(2, 64), _t(66).as_strided((2, 64), (2, 1)))):
        with pytest.raises(RuntimeError, match="gate_add_norm: gate (must be contiguous along columns|is)"):
            call(rows_of, gate=v)
