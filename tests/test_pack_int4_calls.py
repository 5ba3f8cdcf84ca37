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


def test_more_features_than_a_c_int(packed):
    """2^32 + 16 features would be 16 to the C entry; beyond 2^30 every form refuses"""
    for n, k, scales in ((2 ** 32 + 16, 8, 1), (16, 2 ** 32 + 8, 1), (2 ** 30 + 8, 8, 1), (16, 2 ** 30 + 8, 1)):
        q = torch.empty(n, k // 2, dtype=torch.uint8, device="meta")
        with pytest.raises(RuntimeError, match="pack_int4: more than 2\\^30 features"):
            packed(q, torch.empty(n, scales, dtype=torch.bfloat16, device="meta"), group=2 ** 33)


def test_weights_of_more_features_than_a_c_int(monkeypatch):
    """... and a weight put together by hand"""
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_native", type("Declines", (), {"linear_int4": staticmethod(lambda *a: None)}))
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")
    n = 2 ** 32 + 16
    w = ops.Int4Weight(meta(1024, dtype=torch.uint8), meta(1, n), None, n, 128, 128)
    with pytest.raises(RuntimeError, match="linear_int4: more than 2\\^30 features"):
        ops.linear_int4(meta(1, 128), w, out=meta(1, n))


def test_groups_past_a_c_int(packed, monkeypatch):
    """2^32 + 128 elements would be groups of 128 to the C entry, of which the scales have only the first"""
    q = torch.zeros(16, 128, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="pack_int4: group 4294967424 "):
        packed(q, _scales(16), group=2 ** 32 + 128)
    monkeypatch.setattr(ops, "_native", type("Declines", (), {"linear_int4": staticmethod(lambda *a: None)}))
    w = ops.Int4Weight(torch.empty(1024, dtype=torch.uint8), torch.ones(1, 16, dtype=torch.bfloat16), None, 16, 256, 2 ** 32 + 128)
    with pytest.raises(RuntimeError, match="linear_int4: group 4294967424 "):
        ops.linear_int4(torch.zeros(1, 256, dtype=torch.bfloat16), w, out=torch.zeros(1, 16, dtype=torch.bfloat16))
