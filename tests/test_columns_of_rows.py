"""Rows of more columns than a C int holds, without a GPU: 2^32 + 64 columns would be 64 to the C entries."""
import pytest
import torch

from brodiffusion_amd import ops


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.fixture
def python_forms(monkeypatch):
    class Declines:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_native", Declines())


N = 2 ** 32 + 64


@pytest.mark.parametrize("call", [
    lambda: ops.gate_add_norm(_meta(2, N), _meta(2, N)), lambda: ops.gate_add_norm(_meta(N), None), lambda: ops.add_rms_norm(_meta(2, N), None, _meta(N), 1e-6), lambda: ops.quantize_rows_int8(_meta(2, N)),
    lambda: ops.linear_act(_meta(2, N), _meta(8, N)), lambda: ops.linear_act(_meta(2, 64), _meta(N, 64))], ids=["gate_add_norm", "norm alone", "add_rms_norm", "quantize_rows_int8", "in_features", "out_features"])
def test_refused(python_forms, call):
    with pytest.raises(RuntimeError, match="more than 2\\^31 - 1 (columns|rows)"):
        call()
