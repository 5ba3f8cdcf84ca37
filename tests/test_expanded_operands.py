"""Operands whose rows or batch items are one (expanded tensors, stride 0): the C entries take a stride of 0 for dense, so the Python forms refuse them. Without a GPU: the
library is a stand-in that must not be reached."""
import pytest
import torch

from brodiffusion_amd import ops

D = 128


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def _one(*shape, dtype=torch.float16):
    """One item, expanded along the first axis"""
    return _t(1, *shape[1:], dtype=dtype).expand(*shape)


def _rows(b, n, d):
    return _t(b, 1, d).expand(b, n, d)


TABLE = _t(6, 32, dtype=torch.float32)
OFFSETS = torch.tensor([0, 6], dtype=torch.int32)
CALLS = {
    "attention, keys of a batch": lambda: ops.sdpa_forward(_t(2, 6, D), _one(2, 6, D), _t(2, 6, D), 2),
    "attention, values of a batch": lambda: ops.sdpa_forward(_t(2, 6, D), _t(2, 6, D), _one(2, 6, D), 2),
    "attention, query rows": lambda: ops.sdpa_forward(_rows(2, 6, D), _t(2, 6, D), _t(2, 6, D), 2),
    "attention, rows": lambda: ops.flash_attention_forward(_t(6, D), _one(6, D), _t(6, D), None, 2, False),
    "attention, out": lambda: ops.sdpa_forward(_t(2, 6, D), _t(2, 6, D), _t(2, 6, D), 2, out=_one(2, 6, D)),
    "attention, a prefix for all items": lambda: ops.sdpa_forward(_t(2, 6, D), _t(2, 6, D), _t(2, 6, D), 2, k_prefix=_one(2, 5, D), v_prefix=_t(2, 5, D)),
    "attention, logit bias": lambda: ops.sdpa_forward(_t(6, D), _t(6, D), _t(6, D), 2, logit_bias=_one(6, 6, dtype=torch.float32)),
    "packed sequences": lambda: ops.flash_attention_varlen_forward(_t(6, D), _one(6, D), _t(6, D), OFFSETS, OFFSETS, 1, 6, 6, 2, 64, False),
    "packed sequences, out": lambda: ops.flash_attention_varlen_forward(_t(6, D), _t(6, D), _t(6, D), OFFSETS, OFFSETS, 1, 6, 6, 2, 64, False, out=_one(6, D)),
    "row bias": lambda: ops.add_inplace_row_bias(_one(6, D), _t(D)),
    "rope": lambda: ops.rope_apply(_one(6, D), TABLE, TABLE, 64, 2),
    "rope, out": lambda: ops.rope_apply(_t(6, D), TABLE, TABLE, 64, 2, out=_one(6, D)),
    "scaled rows": lambda: ops.scale_rows(_one(6, D)),
    "scaled rows, out": lambda: ops.scale_rows(_t(6, D), out=_one(6, D)),
    "head norm": lambda: ops.headnorm_rope(_one(6, D), _t(64), 1e-6, None, None, 64, 2),
    "head norm, out": lambda: ops.headnorm_rope(_t(6, D), _t(64), 1e-6, None, None, 64, 2, out=_one(6, D)),
    "head norm, cache": lambda: ops.headnorm_rope(_t(6, D), _t(64), 1e-6, None, None, 64, 2, cache_out=_one(4, D)),
    "map": lambda: ops.attention_map_avg(_one(6, D), _t(6, D), _t(12, dtype=torch.float32), 2),
    "map, keys": lambda: ops.attention_map_avg(_t(6, D), _one(6, D), _t(12, dtype=torch.float32), 2),
    "map, out": lambda: ops.attention_map_avg(_t(6, D), _t(6, D), _t(12, dtype=torch.float32), 2, out=_one(6, 6, dtype=torch.float32)),
    "map, logit bias": lambda: ops.attention_map_avg(_t(6, D), _t(6, D), _t(12, dtype=torch.float32), 2, logit_bias=_one(6, 6, dtype=torch.float32)),
    "linear attention": lambda: ops.linear_attention_relu_forward(_t(2, 6, D), _one(2, 6, D), _t(2, 6, D), 4),
    "linear attention, channel-major": lambda: ops.linear_attention_relu_forward_channel_major(_t(2, D, 8), _t(2, D, 8), _one(2, D, 8), 4),
    "row norm": lambda: ops.rms_norm_rows(_one(6, D), _t(D), 1e-6),
    "row norm, out": lambda: ops.rms_norm_rows(_t(6, D), _t(D), 1e-6, out=_one(6, D)),
}


@pytest.fixture
def no_gpu(monkeypatch):
    class Library:
        def __getattr__(self, name):
            def entry(*a):
                assert name.endswith(("_bytes", "_supported")), f"{name} was called"
                return 0
            return entry

    class Declines:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_native", Declines())
    monkeypatch.setattr(ops.capi, "lib", lambda: Library())


@pytest.mark.parametrize("what", list(CALLS))
def test_refused(no_gpu, what):
    with pytest.raises(RuntimeError, match="expanded"):
        CALLS[what]()


def test_one_row_of_any_stride(no_gpu):
    """An axis of one entry has no stride to speak of: such calls go to the library as before"""
    for call in (lambda: ops.rms_norm_rows(_t(D)[None], _t(D), 1e-6), lambda: ops.rms_norm_rows(_one(1, D), _t(D), 1e-6), lambda: ops.scale_rows(_t(1, D).expand(1, D))):
        with pytest.raises(AssertionError, match="was called"):
            call()
