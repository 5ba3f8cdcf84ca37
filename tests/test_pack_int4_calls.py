"""pack_int4's Python form without a GPU: what it hands to the C entry, and what it refuses (the entry is a stand-in that notes its arguments)."""
import pytest
import torch

from brodiffusion_amd import ops


@pytest.fixture
def packed(monkeypatch):
    """pack_int4 on CPU and meta tensors; returns the arguments of the entry, None where it was not reached"""
    got = []

    class Library:
        @staticmethod
        def mi_int4_packed_bytes(n, k):
            return 1024

        @staticmethod
        def mi_pack_int4(args):
            got.append(args._obj)
            return 0
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops.capi, "lib", lambda: Library)

    def call(*args, **kw):
        got.clear()
        ops.pack_int4(*args, **kw)
        return got[0] if got else None
    return call


def _scales(n, groups=1):
    return torch.ones(n, groups, dtype=torch.bfloat16)


def test_row_strides(packed):
    q = torch.zeros(16, 64, dtype=torch.uint8)
    for rows, stride in ((q, 64), (torch.zeros(16, 80, dtype=torch.uint8)[:, :64], 80), (torch.zeros(16, 80, dtype=torch.uint8)[:1, :64], 64)):
        a = packed(rows, _scales(rows.shape[0]))
        assert (a.q, a.out_features, a.in_features, a.q_row_stride) == (rows.data_ptr(), rows.shape[0], 128, stride)


def test_rows_that_are_one(packed):
    """A stride of zero would mean dense rows to the C entry: 16 rows would be read where one is"""
    one = torch.zeros(1, 64, dtype=torch.uint8).expand(16, 64)
    for q in (one, torch.zeros(16 * 32 + 32, dtype=torch.uint8).as_strided((16, 64), (32, 1))):
        with pytest.raises(RuntimeError, match="pack_int4: q must be whole rows apart"):
            packed(q, _scales(16))
